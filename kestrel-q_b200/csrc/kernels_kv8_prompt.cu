// Attention of prompts over the paged 8-bit cache on the 5th-generation tensor
// cores.  (The mathematics and the scaling of the operands: see
// kernels_kv8_attend.cu.)
//
// One CTA takes MT tiles of 128 query rows (request rows r = token * G + head)
// of one key/value head and walks the tokens they see, 128 (or 64) at a time:
//
//   S = Q K^T     tcgen05.mma, Q and the widened keys in shared memory
//   P = weights   TMEM -> registers -> TMEM, over the S they came from
//   O += P V      tcgen05.mma, P from TMEM, the widened values in shared memory
//
// Roles (one CTA per SM):
//   2 MT warpgroups  softmax: two threads share a row, half of a step's tokens
//                    each; two passes over S in TMEM (maximum, weights), the
//                    maxima meet in shared memory
//   2 warpgroups     widening: pages -> registers (the loads of the next keys
//                    or values run while the current ones wait for their slot)
//                    -> fp16 in the 128-byte-swizzled image the MMA reads
//   1 warp           one thread issues the MMAs and owns TMEM
// The inner loops are kept rolled: unrolled to a row of 128 tokens in
// registers, one thread a row, the softmax waited for instructions and took
// 6000 cycles a step (1054 us for an 8k prompt, head dimension 128).
// Registers move between the roles (setmaxnreg) within the launch's total:
// UTile checks the sum.
// With two tiles, one tile's softmax runs under the other's products; with one
// (head dimension 256, or two-term F32 operands), S is double-buffered and the
// next product runs under the softmax.
//
// The weights' token order inside a group of 16 is free (it is summed over),
// and is chosen so that a lane's value codes are 8 contiguous bytes of the
// image.
//
// Every wait is bounded: one that gives up raises the CTA's abort flag, every
// role leaves its loop, MMAs in flight are waited for (bounded) and TMEM is
// freed.
#include "kernels_kv8.cuh"

#include <algorithm>

namespace kqb {

namespace {

constexpr uint32_t kUTmem = 512;
constexpr int kWidenWarps = 8;

// What the roles share besides the operands, behind them in shared memory (in
// dynamic shared memory, so that the operands begin at its start, which is
// 1024-byte aligned: the swizzle's atoms need that).
template <int MT>
struct UShared {
    uint64_t s_full[2], p_full[2], pv_done[2], k_full[2], k_empty[2], v_full[2], v_empty[2], q_full, drained, met[MT];
    uint32_t tmem, gave_up;
    float meet[2][MT][2][128];   // by turn, tile, half: a row's two threads
};

template <int D, int TERMS>
struct UTile {
    static constexpr int MT = D * TERMS <= 128 ? 2 : 1;          // query tiles of 128 rows
    static constexpr int SB = 3 - MT;                            // S buffers per tile
    static constexpr uint32_t rows = 128 * MT;
    static constexpr uint32_t tokens = D == 256 ? 64 : 128;      // per step
    static constexpr uint32_t groups = tokens / kG;
    static constexpr int NK = D * TERMS == 512 ? 1 : 2, NV = 2;  // key slots, value slots
    static constexpr uint32_t q_bytes = rows * D * 2 * TERMS;
    static constexpr uint32_t slot = tokens * D * 2;
    static constexpr uint32_t operands = q_bytes + (NK + NV) * slot, smem = operands + sizeof(UShared<MT>);
    static constexpr uint32_t s_col = MT * D;                    // first S column
    static constexpr int softmax_warps = 8 * MT;
    static constexpr int threads = (softmax_warps + kWidenWarps + 4) * 32;
    // registers a thread: what the launch gives (a multiple of 8), and the roles' shares of it
    static constexpr int launch_regs = 65536 / threads / 8 * 8;
    static constexpr int softmax_regs = MT == 2 ? 80 : 112, widen_regs = MT == 2 ? 64 : 96, mma_regs = 56;
    static constexpr int units = groups * (D / 64) / kWidenWarps;   // (group, 64 features) per widening warp and step
    static constexpr uint32_t flush = 512 / tokens;                 // steps (two-term operands)
    static_assert(s_col + MT * SB * tokens <= kUTmem, "TMEM");
    static_assert(units * kWidenWarps == (int)groups * (D / 64), "units");
    static_assert(2 * MT * softmax_regs + 2 * widen_regs + mma_regs <= (2 * MT + 3) * launch_regs, "registers");
};

// K-major operand in 128-byte-swizzled atoms of 8 rows (1024 bytes): start
// address, stride between atoms, descriptor version 1, swizzle mode 2.
__device__ __forceinline__ uint64_t operand(uint32_t address) {
    return (uint64_t)((address >> 4) & 0x3fffu) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}

// kind::f16: F32 accumulator, fp16 operands, both K-major, M = 128.
constexpr uint32_t instruction(uint32_t n) { return 1u << 4 | (n >> 3) << 17 | (128u >> 4) << 24; }

template <uint32_t N>
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "n"(instruction(N)),
        "r"(accumulate));
}

template <uint32_t N>
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "n"(instruction(N)),
        "r"(accumulate));
}

__device__ __forceinline__ void umma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}

// Ties the loaded registers to the wait, so that no use moves before it.
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}

__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
        "r"(r[30]), "r"(r[31])
        : "memory");
}

// Two F32 values in a register pair, and packed arithmetic on them.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}

__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// A bounded wait of a whole warp: the same answer in every lane.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile uint32_t *quit) {
    return __all_sync(~0u, bar_wait(bar, parity, quit));
}

}  // namespace

// grid (tile, head, split), the last tiles first (they see the most tokens).
template <int D, int TERMS, bool E4M3>
__global__ void __launch_bounds__((UTile<D, TERMS>::threads), 1)
kv8_prompt_kernel(Kv8Cache c, Kv8Step s, Kv8Attend a, Kv8Shape shape, ErrorWord err) {
    using T = UTile<D, TERMS>;
    constexpr int MT = T::MT, NK = T::NK, NV = T::NV;
    constexpr bool BF16 = TERMS == 1;
    extern __shared__ __align__(1024) uint8_t smem[];
    UShared<MT> &sh = *reinterpret_cast<UShared<MT> *>(smem + T::operands);
    uint64_t *const s_full = sh.s_full, *const p_full = sh.p_full, *const pv_done = sh.pv_done, *const k_full = sh.k_full,
                    *const k_empty = sh.k_empty, *const v_full = sh.v_full, *const v_empty = sh.v_empty;
    volatile uint32_t *quit = &sh.gave_up;
    uint8_t *k_slots = smem + T::q_bytes, *v_slots = k_slots + NK * T::slot;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t G = a.query_heads / c.heads;
    const uint32_t split = blockIdx.x % shape.prompt_splits, u = blockIdx.x / shape.prompt_splits;
    const uint32_t head = u % c.heads, t = shape.prompt_tiles - 1 - u / c.heads;

    if (tid == 0) {
        sh.gave_up = smem_u32(smem) % 1024 != 0;   // operands would be misread: give up at once
        for (int i = 0; i < 2; ++i) {
            bar_init(&s_full[i], 1);
            bar_init(&p_full[i], 8);
            bar_init(&pv_done[i], 1);
            bar_init(&k_full[i], kWidenWarps);
            bar_init(&k_empty[i], 1);
            bar_init(&v_full[i], kWidenWarps);
            bar_init(&v_empty[i], 1);
        }
        bar_init(&sh.q_full, 8 * MT);
        for (int i = 0; i < MT; ++i) bar_init(&sh.met[i], 8);
        bar_init(&sh.drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    if (__syncthreads_or(tid == 0 && err_raised(err))) return;
    uint32_t start;
    const uint32_t b = find_request(s, G, T::rows, t, lane, start);
    Request rq;
    if (!load_request(c, s, b, rq, err)) return;
    const uint64_t rows64 = (uint64_t)rq.n * G;
    if (t < start || rows64 <= shape.row_limit || (uint64_t)(t - start) * T::rows >= rows64) return;
    const uint32_t rows = (uint32_t)rows64, row0 = (t - start) * T::rows, row_end = min(row0 + T::rows, rows);
    const uint32_t groups = visible_groups(rq, G, row_end);
    const uint32_t each = split_groups(groups, shape.prompt_groups, shape.prompt_splits, kPromptUnit);
    const uint32_t g0 = split * each, g1 = min(g0 + each, groups);
    if (split > 0 && g0 >= groups) return;
    const uint32_t steps = g1 > g0 ? (g1 - g0 + T::groups - 1) / T::groups : 0u;
    const uint32_t tiles = min((uint32_t)MT, (row_end - row0 + 127) / 128);   // tiles that hold rows
    const int32_t *table = s.table + (uint64_t)b * s.table_stride;
    const uint32_t per_page = c.page_tokens / kG;

    constexpr uint32_t kMmaWarp = T::softmax_warps + kWidenWarps;
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(kUTmem));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem;

    if (warp < T::softmax_warps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T::softmax_regs));
        // ---------------------------------------------------------- softmax
        const uint32_t m = warp >> 3, half = warp >> 2 & 1, row_in = tid & 127, row = row0 + m * 128 + row_in, token_of = row / G;
        const bool live = row < row_end;
        const uint32_t lanes = (warp & 3) << 21;   // the warp's 32 lanes, in bits 16 and up of a TMEM address
        // a value of the row's other thread, for this thread's: both warpgroups
        // of the tile make the same calls (two slots, as a thread may still
        // read the last one's)
        uint32_t meetings = 0;
        bool ok = true;
        auto exchange = [&](float x) {
            const uint32_t parity = meetings++ & 1;
            sh.meet[parity][m][half][row_in] = x;
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.met[m]);
            ok = warp_wait(&sh.met[m], parity, quit);
            return sh.meet[parity][m][half ^ 1][row_in];
        };
        int32_t limit = -1;
        float factor = 0.0f;
        {
            // this thread's half row of Q, scaled and split, into the swizzled image
            constexpr int H = D / 2;
            const uint64_t at = live ? ((uint64_t)rq.first + token_of) * a.q_stride + (uint64_t)(head * G + row % G) * D + half * H : 0;
            float top = 0.0f;
            bool bad = false;
            if (live) {
#pragma unroll 8
                for (int f = 0; f < H; f += 4) {
                    const float4 x = load4<BF16>(a.q, at + f);
                    bad |= !(fabsf(x.x) < INFINITY) || !(fabsf(x.y) < INFINITY) || !(fabsf(x.z) < INFINITY) ||
                           !(fabsf(x.w) < INFINITY);
                    top = fmaxf(fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
                }
                limit = (int32_t)(rq.length - rq.n + token_of);
            }
            if (bad) raise(err, kErrNonFinite);
            top = fmaxf(top, exchange(top));
            // the largest element into [2^13, 2^14); the sign of the softmax
            // scale goes into Q, so that factors are not negative
            const int e = max((int)(__float_as_uint(top) >> 23), 27) - 127 - 13;
            const float up = copysignf(__uint_as_float((uint32_t)(127 - e) << 23), a.scale_log2);
            factor = fabsf(a.scale_log2) * __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll 4
            for (int f = 0; f < H; f += 8) {
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y = x;
                if (live) x = load4<BF16>(a.q, at + f), y = load4<BF16>(a.q, at + f + 4);
                x.x *= up, x.y *= up, x.z *= up, x.w *= up, y.x *= up, y.y *= up, y.z *= up, y.w *= up;
                const uint4 h = make_uint4(pack_half(x.x, x.y), pack_half(x.z, x.w), pack_half(y.x, y.y), pack_half(y.z, y.w));
                const uint32_t g = half * H + f;
                uint8_t *at8 = smem + m * (128 * D * 2 * TERMS) + (g / 64) * 16384 + row_in * 128 + (((g % 64 / 8) ^ (row_in & 7)) << 4);
                *reinterpret_cast<uint4 *>(at8) = h;
                if constexpr (TERMS == 2)
                    *reinterpret_cast<uint4 *>(at8 + 128 * D * 2) =
                        make_uint4(pack_rest(x.x, x.y, h.x), pack_rest(x.z, x.w, h.y), pack_rest(y.x, y.y, h.z),
                                   pack_rest(y.z, y.w, h.w));
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(&sh.q_full);

        float mx = -INFINITY, sum = 0.0f, ref = 0.0f;   // sum: of this thread's tokens
        bool saved = false;     // sums of earlier steps are in the output (or the partials)
        float kept = 1.0f;      // what they are to be multiplied by
        constexpr uint32_t kHalf = T::tokens / 2;
        const uint32_t o_at = tmem + lanes + m * D + half * (D / 2);   // this thread's half of the features
        const bool whole = groups <= each;
        const Partials part(a.workspace + shape.row_floats, (uint64_t)t * c.heads + head, shape.prompt_splits, T::rows, D,
                            (uint64_t)shape.prompt_tiles * c.heads);
        const uint32_t in_tile = m * 128 + row_in, qh = head * G + row % G;
        const uint64_t out_at = ((uint64_t)rq.first + token_of) * a.out_stride + (uint64_t)qh * D + half * (D / 2);
        // O * scale + (what is saved) * keep, into the output or the partials.
        // The accumulators' additions truncate: with two-term operands, whose
        // result is to be good to F32, O goes out and starts anew every 512
        // tokens (prompt chunks over 3000 tokens: error 6.5e-6 without).
        auto move_out = [&](float scale, float keep) {
            bool fine = true;
#pragma unroll 1
            for (int n = 0; n < D / 2; n += 32) {
                uint32_t x[32];
                if (steps > 0) {
                    tmem_load(o_at + n, x);
                    tmem_loaded(x);
                } else {
#pragma unroll
                    for (int k = 0; k < 32; ++k) x[k] = 0;
                }
                if (!live) continue;
                float *to = whole ? static_cast<float *>(a.out) + (BF16 ? 0 : out_at + n)
                                  : part.o + ((uint64_t)split * T::rows + in_tile) * D + half * (D / 2) + n;
#pragma unroll
                for (int g = 0; g < 32; g += 4) {
                    float4 o = make_float4(__uint_as_float(x[g]) * scale, __uint_as_float(x[g + 1]) * scale,
                                           __uint_as_float(x[g + 2]) * scale, __uint_as_float(x[g + 3]) * scale);
                    if (TERMS == 2 && keep != 0.0f) {
                        const float4 y = *reinterpret_cast<const float4 *>(to + g);
                        o.x += y.x * keep, o.y += y.y * keep, o.z += y.z * keep, o.w += y.w * keep;
                    }
                    fine &= fabsf(o.x) + fabsf(o.y) + fabsf(o.z) + fabsf(o.w) < INFINITY;
                    if (BF16 && whole)
                        store4<BF16>(a.out, out_at + n + g, o);
                    else
                        *reinterpret_cast<float4 *>(to + g) = o;
                }
            }
            return fine;
        };
        if (ok && m < tiles) {
            const int32_t all_see = __reduce_min_sync(~0u, limit);   // the last token that every row of the warp sees
            // lane l holds the scales of the step's group l; page ids are read two steps ahead, scales one
            auto page_of = [&](uint32_t j) {
                const uint32_t g = g0 + j * T::groups + lane;
                return lane < T::groups && j < steps && g < g1 ? table[g / per_page] : -1;
            };
            auto scales_of = [&](int32_t id) {   // out of range: the widening warps raise the error
                return id >= 0 && (uint32_t)id < c.pages
                           ? *reinterpret_cast<const float2 *>(c.scales + ((uint64_t)id * c.heads + head) * 2)
                           : make_float2(0.0f, 0.0f);
            };
            float2 next = scales_of(page_of(0));
            int32_t id = page_of(1);
            for (uint32_t j = 0; j < steps; ++j) {
                const float2 sc = next;
                next = scales_of(id);
                id = page_of(j + 2);
                const uint32_t buf = MT == 2 ? m : j & 1, phase = MT == 2 ? j & 1 : j >> 1 & 1;
                const uint32_t s_at = tmem + lanes + T::s_col + buf * T::tokens + half * kHalf;
                const uint32_t group = half * (T::groups / 2);   // this thread's first
                const int32_t token = (int32_t)((g0 + j * T::groups + group) * kG);
                const bool mask = token + (int32_t)kHalf - 1 > all_see;
                ok = warp_wait(&s_full[buf], phase, quit);
                if (!ok) break;
                fence_after();
                // maximum
                float top = -INFINITY, most = sc.y;
#pragma unroll
                for (int o = 1; o < (int)T::groups; o <<= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, o));
                most = __shfl_sync(~0u, most, 0);
#pragma unroll 1
                for (uint32_t q = 0; q < kHalf / 32; ++q) {
                    uint32_t r[32];
                    tmem_load(s_at + q * 32, r);
                    const float f0 = factor * __shfl_sync(~0u, sc.x, group + 2 * q);
                    const float f1 = factor * __shfl_sync(~0u, sc.x, group + 2 * q + 1);
                    tmem_loaded(r);
                    if (mask) {
                        const int32_t seen = limit - token - (int32_t)q * 32;   // tokens 0 .. seen are visible
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (k > seen) r[k] = 0xff800000u;
                    }
                    float x = -INFINITY, y = -INFINITY;
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        x = max3(x, __uint_as_float(r[k]), __uint_as_float(r[k + 1]));
                        y = max3(y, __uint_as_float(r[16 + k]), __uint_as_float(r[17 + k]));
                    }
                    top = max3(top, x * f0, y * f1);   // a factor of 0 times -inf is NaN, which the maximum drops
                }
                top = fmaxf(top, exchange(top));
                if (!ok) break;
                const bool lift = top > mx + kRaise;   // -inf + 8 is -inf: the first finite logit lifts
                float by = 1.0f;
                if (lift) {
                    by = exp2_approx(mx - top);
                    mx = top;
                    sum *= by;
                    kept *= by;
                }
                if (most > ref) {
                    // the next power of two, within the normal range
                    const uint32_t e = min((__float_as_uint(most) + 0x7fffffu) & 0x7f800000u, 0x7f000000u);
                    const float up = __uint_as_float(max(e, 0x00800000u));
                    by *= ref / up;
                    ref = up;
                }
                const bool flush = TERMS == 2 && j > 0 && j % T::flush == 0;
                // O is at rest once the last step's second product is done.  Every
                // step waits for it before it hands its weights over, if not
                // here: a parity wait must not fall two phases behind.
                const bool touch = flush || (j > 0 && __any_sync(~0u, by != 1.0f));
                if (touch) {
                    ok = warp_wait(&pv_done[MT == 2 ? m : 0], (j - 1) & 1, quit);
                    if (!ok) break;
                    fence_after();
                    if (flush) {
                        // by: since the accumulators' scale; kept: since the saved sums'
                        move_out(by * ref * (1.0f / kWeightScale), saved ? kept : 0.0f);
                        saved = true;
                        kept = 1.0f;
                    } else {
#pragma unroll 1
                        for (int n = 0; n < D / 2; n += 32) {
                            uint32_t x[32];
                            tmem_load(o_at + n, x);
                            tmem_loaded(x);
#pragma unroll
                            for (int k = 0; k < 32; ++k) x[k] = __float_as_uint(__uint_as_float(x[k]) * by);
                            tmem_store32(o_at + n, x);
                        }
                    }
                }
                // weights
                const float base = mx == -INFINITY ? 0.0f : mx, inv = ref > 0.0f ? kWeightScale / ref : 0.0f;
                const uint64_t base2 = pack2(-base, -base);
                uint64_t sum2 = 0;
#pragma unroll 1
                for (uint32_t q = 0; q < kHalf / 32; ++q) {
                    uint32_t r[32];
                    tmem_load(s_at + q * 32, r);
                    float f[2], w[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        f[h] = factor * __shfl_sync(~0u, sc.x, group + 2 * q + h);
                        w[h] = inv * __shfl_sync(~0u, sc.y, group + 2 * q + h);
                    }
                    tmem_loaded(r);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint64_t f2 = pack2(f[h], f[h]);
#pragma unroll
                        for (int k = h * 16; k < h * 16 + 16; k += 2) {
                            float x, y;
                            unpack2(fma2(pack2(__uint_as_float(r[k]), __uint_as_float(r[k + 1])), f2, base2), x, y);
                            r[k] = __float_as_uint(exp2_approx(x));
                            r[k + 1] = __float_as_uint(exp2_approx(y));
                        }
                    }
                    if (mask) {
                        const int32_t seen = limit - token - (int32_t)q * 32;
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (k > seen) r[k] = 0;
                    }
                    // pairs of a group in the values' order: (0,1) (8,9) (2,3) (10,11) ...; then the low parts
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const int at = (k >> 3) * 16 + (k & 1) * 8 + (k >> 1 & 3) * 2;
                        const uint64_t e2 = pack2(__uint_as_float(r[at]), __uint_as_float(r[at + 1]));
                        sum2 = add2(sum2, e2);
                        float x, y;
                        unpack2(mul2(e2, pack2(w[k >> 3], w[k >> 3])), x, y);
                        hi[k] = pack_half(x, y);
                        if constexpr (TERMS == 2) lo[k] = pack_rest(x, y, hi[k]);
                    }
                    tmem_store16(s_at + q * 32, hi);
                    if constexpr (TERMS == 2) tmem_store16(s_at + q * 32 + 16, lo);
                }
                float x, y;
                unpack2(sum2, x, y);
                sum += x + y;
                if (j > 0 && !touch) ok = warp_wait(&pv_done[MT == 2 ? m : 0], (j - 1) & 1, quit);
                if (!ok) break;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&p_full[buf]);
            }
            if (ok && steps > 0) ok = warp_wait(&pv_done[MT == 2 ? m : 0], (steps - 1) & 1, quit);
            fence_after();
            if (ok) sum += exchange(sum);
            if (ok) {
                const float norm = whole ? (sum > 0.0f ? 1.0f / sum : 0.0f) : 1.0f;
                const bool fine = move_out(ref * (1.0f / kWeightScale) * norm, saved ? kept * norm : 0.0f);
                if (live) {
                    if (half == 0) {
                        if (!whole)
                            part.ml[in_tile * shape.prompt_splits + split] = make_float2(mx, sum);
                        else if (a.lse != nullptr)
                            a.lse[((uint64_t)rq.first + token_of) * a.query_heads + qh] =
                                sum > 0.0f ? (mx + log2f(sum)) * kLn2 : -INFINITY;
                    }
                    if (whole && (!fine || !(sum < INFINITY))) raise(err, kErrNonFinite);
                }
            }
        }
    } else if (warp < kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::widen_regs));
        // --------------------------------------------------------- widening
        const uint32_t w = warp - T::softmax_warps;
        constexpr int U = T::units;
        const uint64_t page_bytes = 2ull * c.page_tokens * D;
        // lane l: where group l's codes are (UINT64_MAX: behind the last); page ids are read two steps ahead
        auto page_of = [&](uint32_t j) {
            const uint32_t g = g0 + j * T::groups + lane;
            return lane < T::groups && j < steps && g < g1 ? table[g / per_page] : INT32_MIN;
        };
        auto place_of = [&](uint32_t j, int32_t id) {
            if (id == INT32_MIN) return UINT64_MAX;
            const uint32_t g = g0 + j * T::groups + lane;
            const bool in = id >= 0 && (uint32_t)id < c.pages;
            if (!in) raise(err, kErrStep);
            return (uint64_t)(((uint64_t)(in ? id : 0) * c.heads + head) * page_bytes + (uint64_t)(g % per_page) * 32 * D);
        };
        uint64_t place = place_of(0, page_of(0));
        int32_t id = page_of(1);
        constexpr uint32_t kNothing = E4M3 ? 0u : 0x80808080u;
        // two 16-byte pieces of each of this warp's units: (group, 64 features)
        auto load = [&](uint4 (&x)[U][2], uint32_t side) {
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const uint32_t unit = w + k * kWidenWarps, group = unit / (D / 64), j = unit % (D / 64);
                const uint64_t at = __shfl_sync(~0u, place, group);
                if (at != UINT64_MAX) {
                    const uint4 *p = reinterpret_cast<const uint4 *>(c.codes + at + side * 16 * D + j * 1024) + lane;
                    x[k][0] = __ldg(p);
                    x[k][1] = __ldg(p + 32);
                } else {
                    x[k][0] = x[k][1] = make_uint4(kNothing, kNothing, kNothing, kNothing);
                }
            }
        };
        uint4 kx[U][2], vx[U][2];
        bool ok = true;
        if (steps > 0) load(kx, 0);
        for (uint32_t j = 0; j < steps; ++j) {
            const uint32_t slot = j % NK, vslot = j % NV;
            load(vx, 1);
            if (j >= (uint32_t)NK) ok = warp_wait(&k_empty[slot], (j / NK - 1) & 1, quit);
            if (!ok) break;
            // keys: piece h is token 8 h + g, features 16 t .. + 15: two 16-byte chunks of its row
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const uint32_t unit = w + k * kWidenWarps, group = unit / (D / 64), f = unit % (D / 64);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t r = group * 16 + h * 8 + (lane >> 2), t2 = (lane & 3) * 2;
                    uint8_t *at = k_slots + slot * T::slot + f * (T::tokens * 128) + r * 128;
                    uint4 x, y;
                    widen<E4M3>(kx[k][h].x, x.x, x.y);
                    widen<E4M3>(kx[k][h].y, x.z, x.w);
                    widen<E4M3>(kx[k][h].z, y.x, y.y);
                    widen<E4M3>(kx[k][h].w, y.z, y.w);
                    *reinterpret_cast<uint4 *>(at + ((t2 ^ (r & 7)) << 4)) = x;
                    *reinterpret_cast<uint4 *>(at + (((t2 + 1) ^ (r & 7)) << 4)) = y;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(&k_full[slot]);
            place = place_of(j + 1, id);
            id = page_of(j + 2);
            if (j + 1 < steps) load(kx, 0);
            if (j >= (uint32_t)NV) ok = warp_wait(&v_empty[vslot], (j / NV - 1) & 1, quit);
            if (!ok) break;
            // values: word i of piece h is feature 32 h + 4 g + i (a row of the image), tokens 2t, 2t + 1,
            // 2t + 8, 2t + 9: bytes 8 t of the group's 32
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const uint32_t unit = w + k * kWidenWarps, group = unit / (D / 64), f = unit % (D / 64);
                uint8_t *block = v_slots + vslot * T::slot + (group >> 2) * (D * 128);
                const uint32_t chunk = (group & 3) * 2 + (lane >> 1 & 1), half = (lane & 1) * 8;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 &v = vx[k][h];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint2 x;
                        widen<E4M3>(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w, x.x, x.y);
                        const uint32_t n = f * 64 + h * 32 + (lane >> 2) * 4 + i;
                        *reinterpret_cast<uint2 *>(block + n * 128 + ((chunk ^ (n & 7)) << 4) + half) = x;
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(&v_full[vslot]);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::mma_regs));
    }
    if (warp == kMmaWarp && lane == 0) {
        // ------------------------------------------------------------- MMAs
        const uint32_t q_at = smem_u32(smem), k_at = smem_u32(k_slots), v_at = smem_u32(v_slots);
        auto first_product = [&](uint32_t m, uint32_t buf, uint32_t slot) {
            const uint32_t d = tmem + T::s_col + buf * T::tokens;
#pragma unroll
            for (int term = TERMS - 1; term >= 0; --term)
#pragma unroll
                for (int f = 0; f < D / 64; ++f) {
                    const uint64_t qa = operand(q_at + m * (128 * D * 2 * TERMS) + term * (128 * D * 2) + f * 16384);
                    const uint64_t kb = operand(k_at + slot * T::slot + f * (T::tokens * 128));
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        umma_ss<T::tokens>(d, qa + 2 * k, kb + 2 * k, !(term == TERMS - 1 && f == 0 && k == 0));
                }
        };
        auto second_product = [&](uint32_t m, uint32_t buf, uint32_t slot, bool fresh) {
            const uint32_t p = tmem + T::s_col + buf * T::tokens, d = tmem + m * D;
#pragma unroll
            for (uint32_t k = 0; k < T::tokens / 16; ++k) {
                const uint64_t vb = operand(v_at + slot * T::slot + (k / 4) * (D * 128)) + 2 * (k % 4);
#pragma unroll
                for (int term = TERMS - 1; term >= 0; --term)
                    umma_ts<D>(d, p + k / 2 * 32 + term * 16 + k % 2 * 8, vb, !(fresh && k == 0 && term == TERMS - 1));
            }
        };
        bool ok = bar_wait(&sh.q_full, 0, quit);
        if (ok && steps > 0) {
            ok = bar_wait(&k_full[0], 0, quit);
            if (ok) {
                fence_after();
                for (uint32_t m = 0; m < tiles; ++m) {
                    first_product(m, MT == 2 ? m : 0, 0);
                    umma_commit(&s_full[MT == 2 ? m : 0]);
                }
                umma_commit(&k_empty[0]);
            }
            for (uint32_t j = 0; ok && j < steps; ++j) {
                const bool more = j + 1 < steps;
                const uint32_t slot = j % NV, slot1 = (j + 1) % NK;
                const bool fresh = j == 0 || (TERMS == 2 && j % T::flush == 0);
                if constexpr (MT == 2) {
                    for (uint32_t m = 0; ok && m < tiles; ++m) {
                        ok = bar_wait(&p_full[m], j & 1, quit) && (m > 0 || bar_wait(&v_full[slot], j / NV & 1, quit));
                        if (!ok) break;
                        fence_after();
                        second_product(m, m, slot, fresh);
                        umma_commit(&pv_done[m]);
                        if (m + 1 == tiles) umma_commit(&v_empty[slot]);
                        if (more) {
                            // the next S overwrites the weights that the product reads
                            ok = (m > 0 || bar_wait(&k_full[slot1], (j + 1) / NK & 1, quit)) &&
                                 bar_wait(&pv_done[m], j & 1, quit);
                            if (!ok) break;
                            fence_after();
                            first_product(m, m, slot1);
                            umma_commit(&s_full[m]);
                            if (m + 1 == tiles) umma_commit(&k_empty[slot1]);
                        }
                    }
                } else {
                    if (more) {
                        // into the buffer whose weights the last step's product read
                        ok = bar_wait(&k_full[slot1], (j + 1) / NK & 1, quit) &&
                             (j == 0 || bar_wait(&pv_done[0], (j - 1) & 1, quit));
                        if (!ok) break;
                        fence_after();
                        first_product(0, (j + 1) & 1, slot1);
                        umma_commit(&s_full[(j + 1) & 1]);
                        umma_commit(&k_empty[slot1]);
                    }
                    ok = bar_wait(&p_full[j & 1], j >> 1 & 1, quit) && bar_wait(&v_full[slot], j / NV & 1, quit);
                    if (!ok) break;
                    fence_after();
                    second_product(0, j & 1, slot, fresh);
                    umma_commit(&pv_done[0]);
                    umma_commit(&v_empty[slot]);
                }
            }
        }
        // nothing of this CTA's is in flight after this
        umma_commit(&sh.drained);
        bar_wait(&sh.drained, 0, quit);
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (tid == 0 && *quit) raise(err, kErrTimeout);
    if (warp == kMmaWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kUTmem));
    }
}

namespace {

template <int D, int TERMS, bool E4M3>
void launch_prompt(const Kv8Cache &c, const Kv8Step &s, const Kv8Attend &a, const Kv8Shape &h, ErrorWord err,
                   cudaStream_t stream) {
    constexpr uint32_t smem = UTile<D, TERMS>::smem;
    static DeviceOnce once;
    once.run([] {
        cudaFuncSetAttribute(kv8_prompt_kernel<D, TERMS, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    });
    KernelTimer timer("kv8_prompt", stream);
    launch_pdl(kv8_prompt_kernel<D, TERMS, E4M3>, h.prompt_tiles * c.heads * h.prompt_splits, UTile<D, TERMS>::threads, smem, stream, c, s, a, h,
               err);
    count_launch();
}

template <int D>
void launch_prompt_typed(const Kv8Cache &c, const Kv8Step &s, const Kv8Attend &a, const Kv8Shape &h, ErrorWord err,
                         cudaStream_t stream) {
    if (a.bf16)
        c.e4m3 ? launch_prompt<D, 1, true>(c, s, a, h, err, stream) : launch_prompt<D, 1, false>(c, s, a, h, err, stream);
    else
        c.e4m3 ? launch_prompt<D, 2, true>(c, s, a, h, err, stream) : launch_prompt<D, 2, false>(c, s, a, h, err, stream);
}

}  // namespace

uint32_t kv8_prompt_rows(uint32_t dim, bool bf16) {
    if (bf16) return dim == 256 ? UTile<256, 1>::rows : dim == 128 ? UTile<128, 1>::rows : UTile<64, 1>::rows;
    return dim == 256 ? UTile<256, 2>::rows : dim == 128 ? UTile<128, 2>::rows : UTile<64, 2>::rows;
}

void launch_kv8_prompt(const Kv8Cache &c, const Kv8Step &s, const Kv8Attend &a, const Kv8Shape &shape, ErrorWord err,
                       cudaStream_t stream) {
    if (c.dim == 256)
        launch_prompt_typed<256>(c, s, a, shape, err, stream);
    else if (c.dim == 128)
        launch_prompt_typed<128>(c, s, a, shape, err, stream);
    else
        launch_prompt_typed<64>(c, s, a, shape, err, stream);
}

}  // namespace kqb
