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
// Roles (512 threads, one CTA per SM):
//   MT warpgroups  softmax: a thread owns a row, so maxima and sums need no
//                  exchange; two passes over its S in TMEM (maximum, weights)
//   3 - MT         widening: pages -> registers (the loads of the next keys
//   warpgroups     or values run while the current ones wait for their slot)
//                  -> fp16 in the 128-byte-swizzled image the MMA reads
//   1 warp         one thread issues the MMAs and owns TMEM
// With two tiles, one tile's softmax runs under the other's products; with one
// (head dimension 256, or two-term F32 operands), S is double-buffered and the
// next product runs under the softmax.
//
// The weights' token order inside a group of 16 and the values' feature order
// inside 32 are free (both are summed or put back on output), and are chosen
// so that a lane's value codes are 8 contiguous bytes of the image.
//
// Every wait is bounded: one that gives up raises the CTA's abort flag, every
// role leaves its loop, MMAs in flight are waited for (bounded) and TMEM is
// freed.
#include "kernels_kv8.cuh"

#include <algorithm>

namespace kqb {

namespace {

constexpr int kUThreads = 512;
constexpr uint32_t kUTmem = 512;

template <int D, int TERMS>
struct UTile {
    static constexpr int MT = D * TERMS <= 128 ? 2 : 1;          // query tiles of 128 rows
    static constexpr int SB = 3 - MT;                            // S buffers per tile
    static constexpr uint32_t rows = 128 * MT;
    static constexpr uint32_t tokens = D * TERMS == 512 ? 64 : 128;   // per step
    static constexpr uint32_t groups = tokens / kG;
    static constexpr int NK = D == 256 ? 1 : 2;                  // key slots, value slots
    static constexpr int widen_warps = 4 * (3 - MT);
    static constexpr uint32_t q_bytes = rows * D * 2 * TERMS;
    static constexpr uint32_t slot = tokens * D * 2;
    static constexpr uint32_t smem = q_bytes + 2 * NK * slot + 1024;
    static constexpr uint32_t s_col = MT * D;                    // first S column
    static constexpr int units = groups * (D / 64) / widen_warps;   // (group, 64 features) per widening warp and step
    static_assert(s_col + MT * SB * tokens <= kUTmem, "TMEM");
    static_assert(units * widen_warps == (int)groups * (D / 64), "units");
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

__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// A bounded wait of a whole warp: the same answer in every lane.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile uint32_t *quit) {
    return __all_sync(~0u, bar_wait(bar, parity, quit));
}

}  // namespace

// grid (tile, head, split), the last tiles first (they see the most tokens).
template <int D, int TERMS, bool E4M3>
__global__ void __launch_bounds__(kUThreads, 1)
kv8_prompt_kernel(Kv8Cache c, Kv8Step s, Kv8Attend a, Kv8Shape shape, ErrorWord err) {
    using T = UTile<D, TERMS>;
    constexpr int MT = T::MT, NK = T::NK;
    constexpr bool BF16 = TERMS == 1;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t s_full[2], p_full[2], pv_done[2], k_full[2], k_empty[2], v_full[2], v_empty[2], q_full, drained;
    __shared__ uint32_t tmem_slot, gave_up;
    volatile uint32_t *quit = &gave_up;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *k_slots = smem + T::q_bytes, *v_slots = k_slots + NK * T::slot;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t G = a.query_heads / c.heads;
    const uint32_t split = blockIdx.x % shape.prompt_splits, u = blockIdx.x / shape.prompt_splits;
    const uint32_t head = u % c.heads, t = shape.prompt_tiles - 1 - u / c.heads;

    if (tid == 0) {
        gave_up = 0;
        for (int i = 0; i < 2; ++i) {
            bar_init(&s_full[i], 1);
            bar_init(&p_full[i], 4);
            bar_init(&pv_done[i], 1);
            bar_init(&k_full[i], T::widen_warps);
            bar_init(&k_empty[i], 1);
            bar_init(&v_full[i], T::widen_warps);
            bar_init(&v_empty[i], 1);
        }
        bar_init(&q_full, 4 * MT);
        bar_init(&drained, 1);
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

    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(kUTmem));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp < 4 * MT) {
        // ---------------------------------------------------------- softmax
        const uint32_t m = warp >> 2, row_in = tid & 127, row = row0 + m * 128 + row_in, token_of = row / G;
        const bool live = row < row_end;
        const uint32_t lanes = (warp & 3) << 21;   // the warp's 32 lanes, in bits 16 and up of a TMEM address
        int32_t limit = -1;
        float factor = 0.0f;
        {
            // this thread's row of Q, scaled and split, into the swizzled image
            const uint64_t at = live ? (uint64_t)(rq.first + token_of) * a.q_stride + (uint64_t)(head * G + row % G) * D : 0;
            float top = 0.0f;
            bool bad = false;
            if (live) {
#pragma unroll 8
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
#pragma unroll 4
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
        if (lane == 0) bar_arrive(&q_full);

        float mx = -INFINITY, sum = 0.0f, ref = 0.0f;
        const uint32_t o_at = tmem + lanes + m * D;
        bool ok = true;
        if (m < tiles) {
            const int32_t all_see = __reduce_min_sync(~0u, limit);   // the last token that every row of the warp sees
            float2 sc = make_float2(0.0f, 0.0f);                     // lane l: the scales of the step's group l
            auto fetch = [&](uint32_t j) {
                const uint32_t g = g0 + j * T::groups + lane;
                float2 x = make_float2(0.0f, 0.0f);
                if (lane < T::groups && g < g1) {
                    const int32_t id = table[g / per_page];
                    if (id >= 0 && (uint32_t)id < c.pages)   // else: the widening warps raise the error
                        x = *reinterpret_cast<const float2 *>(c.scales + ((uint64_t)id * c.heads + head) * 2);
                }
                return x;
            };
            float2 next = fetch(0);
            for (uint32_t j = 0; j < steps; ++j) {
                sc = next;
                if (j + 1 < steps) next = fetch(j + 1);
                const uint32_t buf = MT == 2 ? m : j & 1, phase = MT == 2 ? j & 1 : j >> 1 & 1;
                const uint32_t s_at = tmem + lanes + T::s_col + buf * T::tokens;
                const int32_t token = (int32_t)((g0 + j * T::groups) * kG);
                const bool mask = token + (int32_t)T::tokens - 1 > all_see;
                ok = warp_wait(&s_full[buf], phase, quit);
                if (!ok) break;
                fence_after();
                // maximum
                float top = -INFINITY;
#pragma unroll
                for (uint32_t q = 0; q < T::tokens / 32; ++q) {
                    uint32_t r[32];
                    tmem_load(s_at + q * 32, r);
                    tmem_loaded(r);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float f = factor * __shfl_sync(~0u, sc.x, q * 2 + h);
                        float x = -INFINITY;
                        if (mask) {
                            const int32_t first = token + (int32_t)(q * 32) + h * 16;
#pragma unroll
                            for (int k = 0; k < 16; ++k)
                                if (first + k <= limit) x = fmaxf(x, __uint_as_float(r[h * 16 + k]));
                            x = first <= limit ? x * f : -INFINITY;
                        } else {
#pragma unroll
                            for (int k = 0; k < 16; ++k) x = fmaxf(x, __uint_as_float(r[h * 16 + k]));
                            x *= f;
                        }
                        top = fmaxf(top, x);
                    }
                }
                const bool lift = top > mx + kRaise;   // -inf + 8 is -inf: the first finite logit lifts
                float most = 0.0f;
#pragma unroll
                for (uint32_t g = 0; g < T::groups; ++g) most = fmaxf(most, __shfl_sync(~0u, sc.y, g));
                float by = 1.0f;
                if (lift) {
                    by = exp2_approx(mx - top);
                    mx = top;
                    sum *= by;
                }
                if (most > ref) {
                    // the next power of two, within the normal range
                    const uint32_t e = min((__float_as_uint(most) + 0x7fffffu) & 0x7f800000u, 0x7f000000u);
                    const float up = __uint_as_float(max(e, 0x00800000u));
                    by *= ref / up;
                    ref = up;
                }
                if (j > 0 && __any_sync(~0u, by != 1.0f)) {
                    // O is at rest once the last step's second product is done
                    const uint32_t last = j - 1;
                    ok = warp_wait(&pv_done[MT == 2 ? m : 0], last & 1, quit);
                    if (!ok) break;
                    fence_after();
#pragma unroll 1
                    for (int n = 0; n < D; n += 32) {
                        uint32_t r[32];
                        tmem_load(o_at + n, r);
                        tmem_loaded(r);
#pragma unroll
                        for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * by);
                        tmem_store32(o_at + n, r);
                    }
                }
                // weights
                const float base = mx == -INFINITY ? 0.0f : mx, inv = ref > 0.0f ? kWeightScale / ref : 0.0f;
#pragma unroll
                for (uint32_t q = 0; q < T::tokens / 32; ++q) {
                    uint32_t r[32];
                    tmem_load(s_at + q * 32, r);
                    tmem_loaded(r);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float f = factor * __shfl_sync(~0u, sc.x, q * 2 + h);
                        const float w = inv * __shfl_sync(~0u, sc.y, q * 2 + h);
                        const int32_t first = token + (int32_t)(q * 32) + h * 16;
                        float part = 0.0f;
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            float e = exp2_approx(fmaf(__uint_as_float(r[h * 16 + k]), f, -base));
                            if (mask) e = first + k <= limit ? e : 0.0f;
                            part += e;
                            r[h * 16 + k] = __float_as_uint(e * w);
                        }
                        sum += part;
                    }
                    // pairs of a group in the values' order: (0,1) (8,9) (2,3) (10,11) ...; then the low parts
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const int at = (k >> 3) * 16 + (k & 1) * 8 + (k >> 1 & 3) * 2;
                        const float x = __uint_as_float(r[at]), y = __uint_as_float(r[at + 1]);
                        hi[k] = pack_half(x, y);
                        if constexpr (TERMS == 2) lo[k] = pack_rest(x, y, hi[k]);
                    }
                    tmem_store16(s_at + q * 32, hi);
                    if constexpr (TERMS == 2) tmem_store16(s_at + q * 32 + 16, lo);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&p_full[buf]);
            }
            if (ok && steps > 0) ok = warp_wait(&pv_done[MT == 2 ? m : 0], (steps - 1) & 1, quit);
            fence_after();
            if (ok) {
                const bool whole = groups <= each;
                const Partials part(a.workspace + shape.row_floats, (uint64_t)t * c.heads + head, shape.prompt_splits, T::rows, D,
                                    (uint64_t)shape.prompt_tiles * c.heads);
                const uint32_t in_tile = m * 128 + row_in;
                const float back = ref * (1.0f / kWeightScale);
                const float scale = whole ? (sum > 0.0f ? back / sum : 0.0f) : back;
                const uint64_t token = rq.first + token_of;
                const uint32_t qh = head * G + row % G;
                bool fine = sum < INFINITY;
#pragma unroll 1
                for (int n = 0; n < D; n += 32) {
                    uint32_t r[32];
                    if (steps > 0) {
                        tmem_load(o_at + n, r);
                        tmem_loaded(r);
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; ++k) r[k] = 0;
                    }
                    if (!live) continue;
#pragma unroll
                    for (int g = 0; g < 8; ++g) {   // column 8 i + g is feature 4 g + i
                        const float4 o = make_float4(__uint_as_float(r[g]) * scale, __uint_as_float(r[8 + g]) * scale,
                                                     __uint_as_float(r[16 + g]) * scale, __uint_as_float(r[24 + g]) * scale);
                        if (whole) {
                            fine &= fabsf(o.x) + fabsf(o.y) + fabsf(o.z) + fabsf(o.w) < INFINITY;
                            store4<BF16>(a.out, token * a.out_stride + (uint64_t)qh * D + n + 4 * g, o);
                        } else {
                            *reinterpret_cast<float4 *>(part.o + ((uint64_t)split * T::rows + in_tile) * D + n + 4 * g) = o;
                        }
                    }
                }
                if (live) {
                    if (!whole)
                        part.ml[in_tile * shape.prompt_splits + split] = make_float2(mx, sum);
                    else if (a.lse != nullptr)
                        a.lse[token * a.query_heads + qh] = sum > 0.0f ? (mx + log2f(sum)) * kLn2 : -INFINITY;
                    if (whole && !fine) raise(err, kErrNonFinite);
                }
            }
        }
    } else if (warp < 12) {
        // --------------------------------------------------------- widening
        const uint32_t w = warp - 4 * MT;
        constexpr int U = T::units;
        const uint64_t page_bytes = 2ull * c.page_tokens * D;
        uint64_t place = 0, next = 0;   // lane l: offset of group l's codes (UINT64_MAX: behind the last)
        auto fetch = [&](uint32_t j) {
            const uint32_t g = g0 + j * T::groups + lane;
            uint64_t x = UINT64_MAX;
            if (lane < T::groups && g < g1) {
                const int32_t id = table[g / per_page];
                const bool in = id >= 0 && (uint32_t)id < c.pages;
                if (!in) raise(err, kErrStep);
                x = ((uint64_t)(in ? id : 0) * c.heads + head) * page_bytes + (uint64_t)(g % per_page) * 32 * D;
            }
            return x;
        };
        constexpr uint32_t kNothing = E4M3 ? 0u : 0x80808080u;
        // two 16-byte pieces of each of this warp's units: (group, 64 features)
        auto load = [&](uint4 (&x)[U][2], uint32_t side) {
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const uint32_t unit = w + k * T::widen_warps, group = unit / (D / 64), j = unit % (D / 64);
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
        place = fetch(0);
        if (steps > 0) load(kx, 0);
        for (uint32_t j = 0; j < steps; ++j) {
            const uint32_t slot = j % NK;
            if (j + 1 < steps) next = fetch(j + 1);
            load(vx, 1);
            if (j >= (uint32_t)NK) ok = warp_wait(&k_empty[slot], (j / NK - 1) & 1, quit);
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
            place = next;
            if (j + 1 < steps) load(kx, 0);
            if (j >= (uint32_t)NK) ok = warp_wait(&v_empty[slot], (j / NK - 1) & 1, quit);
            if (!ok) break;
            // values: word i of piece h is feature 32 h + 4 g + i, tokens 2t, 2t + 1, 2t + 8, 2t + 9: row
            // 8 i + g of the feature block's 32, bytes 8 t of the group's 32
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const uint32_t unit = w + k * T::widen_warps, group = unit / (D / 64), f = unit % (D / 64);
                uint8_t *block = v_slots + slot * T::slot + (group >> 2) * (D * 128);
                const uint32_t chunk = (group & 3) * 2 + (lane >> 1 & 1), half = (lane & 1) * 8;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 &v = vx[k][h];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint2 x;
                        widen<E4M3>(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w, x.x, x.y);
                        const uint32_t n = f * 64 + h * 32 + i * 8 + (lane >> 2);
                        *reinterpret_cast<uint2 *>(block + n * 128 + ((chunk ^ (n & 7)) << 4) + half) = x;
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(&v_full[slot]);
        }
    } else if (warp == 12 && lane == 0) {
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
        bool ok = bar_wait(&q_full, 0, quit);
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
                const uint32_t slot = j % NK, slot1 = (j + 1) % NK;
                if constexpr (MT == 2) {
                    for (uint32_t m = 0; ok && m < tiles; ++m) {
                        ok = bar_wait(&p_full[m], j & 1, quit) && (m > 0 || bar_wait(&v_full[slot], j / NK & 1, quit));
                        if (!ok) break;
                        fence_after();
                        second_product(m, m, slot, j == 0);
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
                    ok = bar_wait(&p_full[j & 1], j >> 1 & 1, quit) && bar_wait(&v_full[slot], j / NK & 1, quit);
                    if (!ok) break;
                    fence_after();
                    second_product(0, j & 1, slot, j == 0);
                    umma_commit(&pv_done[0]);
                    umma_commit(&v_empty[slot]);
                }
            }
        }
        // nothing of this CTA's is in flight after this
        umma_commit(&drained);
        bar_wait(&drained, 0);
        if (*quit) raise(err, kErrTimeout);
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 12) {
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
    launch_pdl(kv8_prompt_kernel<D, TERMS, E4M3>, h.prompt_tiles * c.heads * h.prompt_splits, kUThreads, smem, stream, c, s, a, h,
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
