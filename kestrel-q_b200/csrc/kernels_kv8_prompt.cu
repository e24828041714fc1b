// Attention of prompts over the paged 8-bit cache on the 5th-generation tensor
// cores.  (The mathematics and the scaling of the operands: see
// kernels_kv8_attend.cu.)
//
// One CTA takes MT tiles of 128 query rows (request rows r = token * G + head)
// of one key/value head and walks the tokens they see, 128 or 64 at a time:
//
//   S = Q K^T     tcgen05.mma, Q and the widened keys in shared memory
//   P = weights   TMEM -> registers -> TMEM
//   O += P V      tcgen05.mma, P from TMEM, the widened values in shared memory
//
// Roles (one CTA per SM):
//   MT warpgroups      softmax: a thread owns a row (a step's S sits in its
//                      registers), so maxima and sums need no exchange
//   3 - MT warpgroups  widening: pages -> registers (the loads of the next
//                      keys or values run while the current ones wait for
//                      their slot) -> fp16 in the 128-byte-swizzled image the
//                      MMA reads
//   1 warp             one thread issues the MMAs and owns TMEM
// Loads bypass L1: the operands leave it a few KB, and allocating there took
// bandwidth from the MMA's operands (64-row products at 250 cycles, not 48).
// Registers move between the roles (setmaxnreg) within the launch's total:
// UTile checks the sum.
//
// Bound: the chain softmax -> second product -> first product of a tile; the
// tensor pipe is busy a third of the time.  Measured: an 8k bf16 prompt, 32
// query heads of 128 over int8 pages, 843 us: 652 TFLOP/s of the measured 1662
// (mma.sync tiles: 1843 us); of a step's 6200 cycles a tile spends 3700 in its
// softmax (2000 of them on the weights' exponentials, which both tiles share
// one unit for) and 1900 waiting for its two products.  F32 (two-term operands:
// twice the products), 6 prompt chunks of 64..700 tokens, 16 heads of 256 over
// e4m3 pages: 355 us.
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

// What the roles share besides the operands, behind them in shared memory (in
// dynamic shared memory, so that the operands begin at its start, which is
// 1024-byte aligned: the swizzle's atoms need that).
struct UShared {
    uint64_t s_full[2], s_free[2], p_full[2], pv_done[2];   // by tile
    uint64_t k_full[3], k_empty[3], v_full[3], v_empty[3], q_full, drained, back[2];
    uint32_t tmem, gave_up;
};

template <int D, int TERMS>
struct UTile {
    static constexpr int MT = D * TERMS <= 128 ? 2 : 1;          // query tiles of 128 rows
    static constexpr uint32_t rows = 128 * MT;
    // Two tiles: 128 tokens a step, the weights over the S they came from; one
    // tile's softmax runs under the other's products.  One tile: 64 tokens a
    // step, the weights in two buffers of their own, so that S is free as soon
    // as it is in registers and the next product runs under the softmax.
    static constexpr bool alias = MT == 2;
    static constexpr uint32_t tokens = alias ? 128 : 64;         // per step
    static constexpr uint32_t groups = tokens / kG;
    static constexpr int NK = D * TERMS == 512 ? 1 : D == 256 || alias ? 2 : 3;   // key and value slots
    static constexpr int NV = D * TERMS == 512 || alias ? 2 : 3;
    static constexpr uint32_t q_bytes = rows * D * 2 * TERMS;
    static constexpr uint32_t slot = tokens * D * 2;
    static constexpr uint32_t operands = q_bytes + (NK + NV) * slot, smem = operands + sizeof(UShared);
    // TMEM columns: O of each tile, then per tile S and the weights (tokens / 2
    // columns a term)
    static constexpr uint32_t s_col = MT * D, p_cols = tokens / 2 * TERMS, tile_cols = alias ? tokens : tokens + 2 * p_cols;
    static constexpr int softmax_warps = 4 * MT, widen_warps = 4 * (3 - MT);
    static constexpr int threads = 512, launch_regs = 128;
    static constexpr int softmax_regs = MT == 2 ? 184 : 168, widen_regs = MT == 2 ? 96 : 104, mma_regs = 48;
    static constexpr int units = groups * (D / 64) / widen_warps;   // (group, 64 features) per widening warp and step
    static constexpr uint32_t flush = 512 / tokens;                 // steps (two-term operands)
    static_assert(s_col + MT * tile_cols <= kUTmem, "TMEM");
    static_assert(units * widen_warps == (int)groups * (D / 64), "units");
    static_assert(softmax_warps + widen_warps + 4 == threads / 32 && p_cols <= (alias ? tokens : 2 * tokens), "roles");
    static_assert(MT * softmax_regs + widen_warps / 4 * widen_regs + mma_regs <= threads / 128 * launch_regs, "registers");
    static_assert(smem <= 227 * 1024, "shared memory");
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

__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}

__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

}  // namespace

// grid (tile, head, split), the last tiles first (they see the most tokens).
template <int D, int TERMS, bool E4M3>
__global__ void __launch_bounds__((UTile<D, TERMS>::threads), 1)
kv8_prompt_kernel(Kv8Cache c, Kv8Step s, Kv8Attend a, Kv8Shape shape, ErrorWord err) {
    using T = UTile<D, TERMS>;
    constexpr int MT = T::MT, NK = T::NK, NV = T::NV;
    constexpr bool BF16 = TERMS == 1;
    extern __shared__ __align__(1024) uint8_t smem[];
    UShared &sh = *reinterpret_cast<UShared *>(smem + T::operands);
    uint64_t *const pv_done = sh.pv_done, *const k_full = sh.k_full, *const k_empty = sh.k_empty, *const v_full = sh.v_full,
                    *const v_empty = sh.v_empty;
    volatile uint32_t *quit = &sh.gave_up;
    uint8_t *k_slots = smem + T::q_bytes, *v_slots = k_slots + NK * T::slot;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t G = a.query_heads / c.heads;
    const uint32_t split = blockIdx.x % shape.prompt_splits, u = blockIdx.x / shape.prompt_splits;
    const uint32_t head = u % c.heads, t = shape.prompt_tiles - 1 - u / c.heads;

    if (tid == 0) {
        sh.gave_up = smem_u32(smem) % 1024 != 0;   // operands would be misread: give up at once
        for (int m = 0; m < 2; ++m) {
            bar_init(&pv_done[m], 1);
            bar_init(&sh.back[m], 4);
            bar_init(&sh.s_full[m], 1);
            bar_init(&sh.s_free[m], 4);
            bar_init(&sh.p_full[m], 4);
        }
        for (int i = 0; i < 3; ++i) {
            bar_init(&k_full[i], T::widen_warps);
            bar_init(&k_empty[i], 1);
            bar_init(&v_full[i], T::widen_warps);
            bar_init(&v_empty[i], 1);
        }
        bar_init(&sh.q_full, 4 * MT);
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
    const uint32_t page_shift = __ffs(c.page_tokens / kG) - 1;   // groups of a page, a power of two

    constexpr uint32_t kMmaWarp = T::softmax_warps + T::widen_warps;
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
        const uint32_t m = warp >> 2, row_in = tid & 127, row = row0 + m * 128 + row_in, token_of = row / G;
        const bool live = row < row_end;
        const uint32_t lanes = (warp & 3) << 21;   // the warp's 32 lanes, in bits 16 and up of a TMEM address
        int32_t limit = -1;
        float factor = 0.0f;
        {
            // this thread's row of Q, scaled and split, into the swizzled image
            const uint64_t at = live ? ((uint64_t)rq.first + token_of) * a.q_stride + (uint64_t)(head * G + row % G) * D : 0;
            float top = 0.0f;
            bool bad = false;
            if (live) {
#pragma unroll 16
                for (int f = 0; f < D; f += 4) {
                    const float4 x = load4<BF16>(a.q, at + f);
                    bad |= !(fabsf(x.x) < INFINITY) || !(fabsf(x.y) < INFINITY) || !(fabsf(x.z) < INFINITY) ||
                           !(fabsf(x.w) < INFINITY);
                    top = fmaxf(fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
                }
                limit = (int32_t)(rq.length - rq.n + token_of);
            }
            if (bad) raise(err, kErrNonFinite);
            // the largest element into [2^13, 2^14); the sign of the softmax
            // scale goes into Q, so that factors are not negative
            const int e = max((int)(__float_as_uint(top) >> 23), 27) - 127 - 13;
            const float up = copysignf(__uint_as_float((uint32_t)(127 - e) << 23), a.scale_log2);
            factor = fabsf(a.scale_log2) * __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll 8
            for (int f = 0; f < D; f += 8) {
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y = x;
                if (live) x = load4<BF16>(a.q, at + f), y = load4<BF16>(a.q, at + f + 4);
                x.x *= up, x.y *= up, x.z *= up, x.w *= up, y.x *= up, y.y *= up, y.z *= up, y.w *= up;
                const uint4 h = make_uint4(pack_half(x.x, x.y), pack_half(x.z, x.w), pack_half(y.x, y.y), pack_half(y.z, y.w));
                uint8_t *at8 = smem + m * (128 * D * 2 * TERMS) + (f / 64) * 16384 + row_in * 128 + (((f % 64 / 8) ^ (row_in & 7)) << 4);
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

        float mx = -INFINITY, z = -INFINITY, sum = 0.0f;   // reference points: mx of logits, mx + z of O
        const uint32_t o_at = tmem + lanes + m * D;
        const bool whole = groups <= each;
        const Partials part(a.workspace + shape.row_floats, (uint64_t)t * c.heads + head, shape.prompt_splits, T::rows, D,
                            (uint64_t)shape.prompt_tiles * c.heads);
        const uint32_t in_tile = m * 128 + row_in;
        // where row r of this tile goes
        auto row_out = [&](uint32_t r) {
            return whole ? ((uint64_t)rq.first + r / G) * a.out_stride + (uint64_t)(head * G + r % G) * D
                         : (uint64_t)split * T::rows * D + (uint64_t)(r - row0) * D;
        };
        float *const out32 = whole ? static_cast<float *>(a.out) : part.o;
        // Sums of earlier steps (TERMS == 2).  The accumulators' additions
        // truncate; with two-term operands, whose result is to be good to F32,
        // O goes out and starts anew every 512 tokens (prompt chunks over 3000
        // tokens: error 6.5e-6 without, 1.5e-6 with).  It goes to the tile's own
        // output rows (or partials), as long as they are not final: where all
        // 128 rows exist, value 4 f .. 4 f + 3 of row r is the (128 f + r)-th 16
        // bytes of the rows one after another, so that a warp writes 512
        // contiguous bytes; in a tile's rest, in its row.
        bool saved = false;
        float kept = 1.0f;      // what the saved sums are to be multiplied by (they are in O's unit, far from overflow)
        const bool full_tile = row0 + m * 128 + 128 <= row_end;
        auto save = [&](float scale, float keep, bool final_to_tmem) {
            constexpr uint32_t Q = D / 4, kRowsOn = 128 / Q;   // pieces in a row; rows from piece f to piece f + 1 of a thread
            const uint32_t first = row0 + m * 128 + row_in / Q;
            float *to = out32 + (full_tile ? row_out(first) + row_in % Q * 4 : row_out(row));
            uint32_t in_group = first % G;
            const int64_t wrap = whole ? (int64_t)a.out_stride - (int64_t)G * D : 0;
#pragma unroll 1
            for (int n = 0; n < D; n += 32) {
                uint32_t x[32];
                float *at[8];
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    at[g] = to;
                    if (full_tile) {
                        to += kRowsOn * D;
                        for (in_group += kRowsOn; in_group >= G; in_group -= G) to += wrap;
                    } else {
                        to += 4;
                    }
                }
                tmem_load(o_at + n, x);
                float4 y[8];
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    y[g] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (keep != 0.0f && live) y[g] = __ldcg(reinterpret_cast<const float4 *>(at[g]));
                }
                tmem_loaded(x);
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    const float4 o = make_float4(__uint_as_float(x[4 * g]) * scale + y[g].x * keep,
                                                 __uint_as_float(x[4 * g + 1]) * scale + y[g].y * keep,
                                                 __uint_as_float(x[4 * g + 2]) * scale + y[g].z * keep,
                                                 __uint_as_float(x[4 * g + 3]) * scale + y[g].w * keep);
                    x[4 * g] = __float_as_uint(o.x), x[4 * g + 1] = __float_as_uint(o.y);
                    x[4 * g + 2] = __float_as_uint(o.z), x[4 * g + 3] = __float_as_uint(o.w);
                    if (!final_to_tmem && live) __stcg(reinterpret_cast<float4 *>(at[g]), o);
                }
                if (final_to_tmem) tmem_store32(o_at + n, x);
            }
        };
        bool ok = true;
        if (m < tiles) {
            const int32_t all_see = __reduce_min_sync(~0u, limit);   // the last token that every row of the warp sees
            // lane l holds the scales of the step's group l; page ids are read two steps ahead, scales one
            auto page_of = [&](uint32_t j) {
                const uint32_t g = g0 + j * T::groups + lane;
                return lane < T::groups && j < steps && g < g1 ? table[g >> page_shift] : -1;
            };
            auto scales_of = [&](int32_t id) {   // out of range: the widening warps raise the error
                return id >= 0 && (uint32_t)id < c.pages
                           ? *reinterpret_cast<const float2 *>(c.scales + ((uint64_t)id * c.heads + head) * 2)
                           : make_float2(0.0f, 0.0f);
            };
            float2 next = scales_of(page_of(0));
            int32_t id = page_of(1);
#pragma unroll 1
            for (uint32_t j = 0; j < steps; ++j) {
                const float2 sc = next;
                next = scales_of(id);
                id = page_of(j + 2);
                const uint32_t s_at = tmem + lanes + T::s_col + m * T::tile_cols, p_at = T::alias ? s_at : s_at + T::tokens + (j & 1) * T::p_cols;
                const int32_t token = (int32_t)((g0 + j * T::groups) * kG);
                const float size = size_of(sc.y);
                float f[T::groups], w[T::groups], lw[T::groups];
#pragma unroll
                for (uint32_t g = 0; g < T::groups; ++g) {
                    f[g] = factor * __shfl_sync(~0u, sc.x, g);
                    w[g] = __shfl_sync(~0u, sc.y, g);
                    lw[g] = __shfl_sync(~0u, size, g);
                }
                ok = bar_wait_warp(&sh.s_full[m], j & 1, quit);
                if (!ok) break;
                fence_after();
                uint32_t r[T::tokens / 32][32];
#pragma unroll
                for (uint32_t q = 0; q < T::tokens / 32; ++q) tmem_load(s_at + q * 32, r[q]);
#pragma unroll
                for (uint32_t q = 0; q < T::tokens / 32; ++q) tmem_loaded(r[q]);
                if constexpr (!T::alias) {
                    fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&sh.s_free[m]);
                }
                if (token + (int32_t)T::tokens - 1 > all_see) {
                    const int32_t seen = limit - token;   // tokens 0 .. seen are visible
                    asm volatile("");   // a branch, not instructions that every step executes under a predicate
#pragma unroll
                    for (int k = 0; k < (int)T::tokens; ++k)
                        if (k > seen) r[k / 32][k % 32] = 0xff800000u;
                }
                float top = -INFINITY, high[T::groups];
#pragma unroll
                for (uint32_t g = 0; g < T::groups; ++g) high[g] = -INFINITY;
#pragma unroll
                for (int k = 0; k < 16; k += 2)
#pragma unroll
                    for (uint32_t g = 0; g < T::groups; ++g)
                        high[g] = max3(high[g], __uint_as_float(r[g / 2][g % 2 * 16 + k]), __uint_as_float(r[g / 2][g % 2 * 16 + k + 1]));
#pragma unroll
                for (uint32_t g = 0; g < T::groups; ++g) {
                    // a factor of 0 (a zero page) would make -inf NaN
                    if (f[g] == 0.0f) f[g] = 1.0e-38f;
                    high[g] *= f[g];
                    top = fmaxf(top, high[g]);
                }
                // The weights' exponents come from one fused multiply and add each,
                // whose product is not rounded as `top` is: a difference that
                // counts from logits of 2^24 on.  There the products are rounded
                // first.  (The branch takes 12 us of an 8k bf16 prompt's 839; behind
                // the lifts, with the products divided by their factors, 25.)
                if (__any_sync(~0u, fabsf(top) > 0x1p20f && top > -INFINITY)) {
                    asm volatile("");   // a branch
#pragma unroll
                    for (uint32_t k = 0; k < T::tokens; ++k) r[k / 32][k % 32] = __float_as_uint(__uint_as_float(r[k / 32][k % 32]) * f[k / 16]);
#pragma unroll
                    for (uint32_t g = 0; g < T::groups; ++g) f[g] = 1.0f;
                }
                float by = 1.0f;
                if (top > mx + kRaise) {   // -inf + 8 is -inf: the first finite logit lifts
                    const float to = ceilf(top), less = mx - to, l_by = exp2_approx(less);
                    mx = to;
                    z += less;
                    sum *= l_by;
                }
                float top_o = -INFINITY;   // (a row that has seen nothing: NaNs, which the maximum drops)
#pragma unroll
                for (uint32_t g = 0; g < T::groups; ++g) top_o = fmaxf(top_o, high[g] - mx + lw[g]);
                if (top_o > z + kRaise) {
                    const float to = ceilf(top_o);
                    by = exp2_approx(z - to);
                    kept *= by;
                    z = to;
                }
                const bool flush = TERMS == 2 && j > 0 && j % T::flush == 0;
                // O is at rest once the last step's second product is done.  Every
                // step waits for it before it hands its weights over, if not
                // here: a parity wait must not fall two phases behind, and the
                // buffer that these weights go into is free since the last wait.
                const bool touch = flush || (j > 0 && __any_sync(~0u, by != 1.0f));
                if (touch) {
                    ok = bar_wait_warp(&pv_done[m], (j - 1) & 1, quit);
                    if (!ok) break;
                    fence_after();
                    if (flush) {
                        // by: since the accumulators' reference point; kept: since the saved sums'
                        if constexpr (TERMS == 2) save(by, saved ? kept : 0.0f, false);
                        saved = true;
                        kept = 1.0f;
                    } else {
#pragma unroll 1
                        for (int n = 0; n < D; n += 32) {
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
                const float base = mx == -INFINITY ? 0.0f : mx, inv = weight_of(mx, z);
#pragma unroll
                for (uint32_t g = 0; g < T::groups; ++g) w[g] = fminf(w[g] * inv, kMost);
                const uint64_t base2 = pack2(-base, -base);
                uint64_t sum2[2] = {0, 0};
#pragma unroll
                for (uint32_t q = 0; q < T::tokens / 32; ++q) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint64_t f2 = pack2(f[2 * q + h], f[2 * q + h]);
#pragma unroll
                        for (int k = h * 16; k < h * 16 + 16; k += 2) {
                            float x, y;
                            unpack2(fma2(pack2(__uint_as_float(r[q][k]), __uint_as_float(r[q][k + 1])), f2, base2), x, y);
                            r[q][k] = __float_as_uint(exp2_approx(x));
                            r[q][k + 1] = __float_as_uint(exp2_approx(y));
                        }
                    }
                    // pairs of a group in the values' order: (0,1) (8,9) (2,3) (10,11) ...; then the low parts
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const int at = (k >> 3) * 16 + (k & 1) * 8 + (k >> 1 & 3) * 2;
                        const uint64_t e2 = pack2(__uint_as_float(r[q][at]), __uint_as_float(r[q][at + 1]));
                        sum2[k & 1] = add2(sum2[k & 1], e2);
                        const float v = w[2 * q + (k >> 3)];
                        float x, y;
                        unpack2(mul2(e2, pack2(v, v)), x, y);
                        hi[k] = pack_half(x, y);
                        if constexpr (TERMS == 2) lo[k] = pack_rest(x, y, hi[k]);
                    }
                    tmem_store16(p_at + q * 16, hi);
                    if constexpr (TERMS == 2) tmem_store16(p_at + T::tokens / 2 + q * 16, lo);
                }
                float x, y;
                unpack2(add2(sum2[0], sum2[1]), x, y);
                sum += x + y;
                if (j > 0 && !touch) ok = bar_wait_warp(&pv_done[m], (j - 1) & 1, quit);
                if (!ok) break;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.p_full[m]);
            }
            if (ok && steps > 0) ok = bar_wait_warp(&pv_done[m], (steps - 1) & 1, quit);
            fence_after();
            float scale = back_of(mx, z);
            if (TERMS == 2 && ok && saved) {
                // the saved sums come back into TMEM before any row is final
                save(1.0f, kept, true);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.back[m]);
                ok = bar_wait_warp(&sh.back[m], 0, quit);
            }
            if (ok) {
                // to units of 2^m, then by the sum: in one factor, except where that
                // would leave F32's normal numbers (small values)
                float inv = !whole ? 1.0f : sum > 0.0f ? 1.0f / sum : 0.0f;
                if (z > -64.0f) scale *= inv, inv = 1.0f;
                bool fine = sum < INFINITY;
                const uint64_t to = row_out(row);
#pragma unroll 1
                for (int n = 0; n < D; n += 32) {
                    uint32_t x[32];
                    if (steps > 0) {
                        tmem_load(o_at + n, x);
                        tmem_loaded(x);
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; ++k) x[k] = 0;
                    }
                    if (!live) continue;
#pragma unroll
                    for (int g = 0; g < 32; g += 4) {
                        const float4 o = make_float4(__uint_as_float(x[g]) * scale * inv, __uint_as_float(x[g + 1]) * scale * inv,
                                                     __uint_as_float(x[g + 2]) * scale * inv, __uint_as_float(x[g + 3]) * scale * inv);
                        fine &= fabsf(o.x) + fabsf(o.y) + fabsf(o.z) + fabsf(o.w) < INFINITY;
                        if (whole)
                            store4<BF16>(a.out, to + n + g, o);
                        else
                            *reinterpret_cast<float4 *>(out32 + to + n + g) = o;
                    }
                }
                if (live) {
                    if (!whole)
                        part.ml[in_tile * shape.prompt_splits + split] = make_float2(mx, sum);
                    else if (a.lse != nullptr)
                        a.lse[((uint64_t)rq.first + token_of) * a.query_heads + head * G + row % G] =
                            sum > 0.0f ? (mx + log2f(sum)) * kLn2 : -INFINITY;
                    if (whole && !fine) raise(err, kErrNonFinite);
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
            return lane < T::groups && j < steps && g < g1 ? table[g >> page_shift] : INT32_MIN;
        };
        auto place_of = [&](uint32_t j, int32_t id) {
            if (id == INT32_MIN) return UINT64_MAX;
            const uint32_t g = g0 + j * T::groups + lane;
            const bool in = id >= 0 && (uint32_t)id < c.pages;
            if (!in) raise(err, kErrStep);
            return (uint64_t)(((uint64_t)(in ? id : 0) * c.heads + head) * page_bytes + (uint64_t)(g & ((1u << page_shift) - 1)) * 32 * D);
        };
        uint64_t place = place_of(0, page_of(0));
        int32_t id = page_of(1);
        constexpr uint32_t kNothing = E4M3 ? 0u : 0x80808080u;
        // two 16-byte pieces of each of this warp's units: (group, 64 features)
        auto load = [&](uint4 (&x)[U][2], uint32_t side) {
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const uint32_t unit = w + k * T::widen_warps, group = unit / (D / 64), j = unit % (D / 64);
                const uint64_t at = __shfl_sync(~0u, place, group);
                if (at != UINT64_MAX) {
                    const uint4 *p = reinterpret_cast<const uint4 *>(c.codes + at + side * 16 * D + j * 1024) + lane;
                    x[k][0] = __ldcg(p);
                    x[k][1] = __ldcg(p + 32);
                } else {
                    x[k][0] = x[k][1] = make_uint4(kNothing, kNothing, kNothing, kNothing);
                }
            }
        };
        uint4 kx[U][2], vx[U][2];
        bool ok = true;
        uint32_t slot = 0, k_phase = 1, vslot = 0, v_phase = 1;   // a slot's first wait is for no phase: it is free
        if (steps > 0) load(kx, 0);
#pragma unroll 1
        for (uint32_t j = 0; j < steps; ++j) {
            load(vx, 1);
            if (j >= (uint32_t)NK) ok = bar_wait_warp(&k_empty[slot], k_phase, quit);
            if (!ok) break;
            // keys: piece h is token 8 h + g, features 16 t .. + 15: two 16-byte chunks of its row
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const uint32_t unit = w + k * T::widen_warps, group = unit / (D / 64), f = unit % (D / 64);
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
            if (++slot == NK) slot = 0, k_phase ^= 1;
            place = place_of(j + 1, id);
            id = page_of(j + 2);
            if (j + 1 < steps) load(kx, 0);
            if (j >= (uint32_t)NV) ok = bar_wait_warp(&v_empty[vslot], v_phase, quit);
            if (!ok) break;
            // values: word i of piece h is feature 32 h + 4 g + i (a row of the image), tokens 2t, 2t + 1,
            // 2t + 8, 2t + 9: bytes 8 t of the group's 32
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const uint32_t unit = w + k * T::widen_warps, group = unit / (D / 64), f = unit % (D / 64);
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
            if (++vslot == NV) vslot = 0, v_phase ^= 1;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::mma_regs));
    }
    if (warp == kMmaWarp && lane == 0) {
        // ------------------------------------------------------------- MMAs
        const uint32_t q_at = smem_u32(smem), k_at = smem_u32(k_slots), v_at = smem_u32(v_slots);
        // Rolled loops: this thread's instructions are fetched anew every step,
        // and unrolled they took longer than the products (descriptors count 16
        // bytes).
        const uint64_t q_desc = operand(q_at), k_desc = operand(k_at), v_desc = operand(v_at);
        auto first_product = [&](uint32_t m, uint32_t slot) {
            const uint32_t d = tmem + T::s_col + m * T::tile_cols;
            uint32_t more = 0;
            // low parts first: on a sum that is still small, additions that truncate lose little
#pragma unroll 1
            for (int term = TERMS - 1; term >= 0; --term) {
                uint64_t qa = q_desc + (m * TERMS + term) * (128 * D / 8);
                uint64_t kb = k_desc + slot * (T::slot / 16);
#pragma unroll 2
                for (int f = 0; f < D / 64; ++f, qa += 1024, kb += T::tokens * 8) {
                    umma_ss<T::tokens>(d, qa, kb, more);
                    umma_ss<T::tokens>(d, qa + 2, kb + 2, 1);
                    umma_ss<T::tokens>(d, qa + 4, kb + 4, 1);
                    umma_ss<T::tokens>(d, qa + 6, kb + 6, 1);
                    more = 1;
                }
            }
        };
        auto second_product = [&](uint32_t m, uint32_t buf, uint32_t slot, bool fresh) {
            const uint32_t d = tmem + m * D;
            uint32_t more = !fresh;
#pragma unroll 1
            for (int term = TERMS - 1; term >= 0; --term) {
                uint32_t p = tmem + T::s_col + m * T::tile_cols + (T::alias ? 0 : T::tokens + buf * T::p_cols) + term * (T::tokens / 2);
                uint64_t vb = v_desc + slot * (T::slot / 16);
#pragma unroll 1
                for (uint32_t block = 0; block < T::tokens / 64; ++block, p += 32, vb += D * 8) {
                    umma_ts<D>(d, p, vb, more);
                    umma_ts<D>(d, p + 8, vb + 2, 1);
                    umma_ts<D>(d, p + 16, vb + 4, 1);
                    umma_ts<D>(d, p + 24, vb + 6, 1);
                    more = 1;
                }
            }
        };
        bool ok = bar_wait(&sh.q_full, 0, quit);
        uint32_t k_slot = 0, k_phase = 0, v_slot = 0, v_phase = 0;
        auto next_k = [&] {
            umma_commit(&k_empty[k_slot]);
            if (++k_slot == NK) k_slot = 0, k_phase ^= 1;
        };
        auto next_v = [&] {
            umma_commit(&v_empty[v_slot]);
            if (++v_slot == NV) v_slot = 0, v_phase ^= 1;
        };
#pragma unroll 1
        for (uint32_t j = 0; ok && j <= steps; ++j) {
            const uint32_t i = j - 1;
            const bool fresh = i == 0 || (TERMS == 2 && i % T::flush == 0);
            if constexpr (T::alias) {
                // tile by tile: the second product of step j - 1, then the first
                // of step j over the weights that it read
#pragma unroll 1
                for (uint32_t m = 0; m < tiles; ++m) {
                    if (j > 0) {
                        ok = (m > 0 || bar_wait(&v_full[v_slot], v_phase, quit)) && bar_wait(&sh.p_full[m], i & 1, quit);
                        if (!ok) break;
                        fence_after();
                        second_product(m, 0, v_slot, fresh);
                        umma_commit(&pv_done[m]);
                    }
                    if (j < steps) {
                        ok = (m > 0 || bar_wait(&k_full[k_slot], k_phase, quit)) && (j == 0 || bar_wait(&pv_done[m], i & 1, quit));
                        if (!ok) break;
                        fence_after();
                        first_product(m, k_slot);
                        umma_commit(&sh.s_full[m]);
                    }
                }
                if (j > 0) next_v();
                if (j < steps) next_k();
            } else {
                // the first product of step j, once the softmax holds step j - 1's
                if (j < steps) {
                    ok = bar_wait(&k_full[k_slot], k_phase, quit) && (j == 0 || bar_wait(&sh.s_free[0], i & 1, quit));
                    if (!ok) break;
                    fence_after();
                    first_product(0, k_slot);
                    umma_commit(&sh.s_full[0]);
                    next_k();
                }
                // the second product of step j - 1
                if (j > 0) {
                    ok = bar_wait(&v_full[v_slot], v_phase, quit) && bar_wait(&sh.p_full[0], i & 1, quit);
                    if (!ok) break;
                    fence_after();
                    second_product(0, i & 1, v_slot, fresh);
                    umma_commit(&pv_done[0]);
                    next_v();
                }
            }
        }
        // nothing of this CTA's is in flight after this; the abort flag does not
        // cut this wait short
        umma_commit(&sh.drained);
        if (!bar_wait(&sh.drained, 0)) *quit = 1;
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
