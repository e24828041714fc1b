// Causal grouped-query attention over the paged 8-bit cache.
//
//   l_rj = scale * q_r . (sK_j k_j),  j <= position of row r's token
//   out_r = sum_j p_rj sV_j v_j,  p = softmax(l);  lse_r = log sum_j exp l_rj
//
// k, v are the stored codes, sK, sV the scales of j's page and head.  The
// query heads of one key/value head share its codes, so a request's rows
// (token, head of the group) are numbered r = token * G + head and cut into
// tiles that read the same codes.
//
// Products.  Codes convert to fp16 exactly (int8: |code| <= 127; e4m3: 4
// significant bits, exponents -9..8), so the products run on
// mma.sync.m16n8k16 with fp16 operands and F32 accumulators: S = Q K^T with
// rows of Q as the M side, O = P V with the S accumulators as its A operand.
// A row of Q is scaled by an exact power of two so that its largest element
// lies in [2^13, 2^14): bfloat16 queries are then exact in fp16 (elements
// 2^-27 below the row's largest lose bits, below F32's own rounding of the
// sum), F32 queries are split into two fp16 parts (22 bits).  P sV is scaled
// into fp16's range the same way (below) and split in two for F32 outputs;
// for bfloat16 outputs one part is kept: 11 bits, 2^-12 relative per weight
// against the output's own 2^-9.  The page scales multiply the accumulators
// (sK) and the weights (sV), never the codes.
//
// Softmax in base 2, one pass: the reference point m of a row is raised only
// when a logit exceeds it by more than 8, so weights stay below 2^8 and the
// accumulators are rarely rescaled; m, the sums l and O are F32.  The weights
// entering the second product are p * sV / R * 2^6 with R the smallest power
// of two not below any sV seen (O is rescaled exactly when R grows): at most
// 2^14, and anything below 2^-24 of that is lost (2^-38 of the largest).
//
// Layout.  A page keeps its codes in the order the fragments need (see
// Kv8Cache), so a warp reads both operands with conflict-free 16-byte shared
// loads and no transposes, and a group of 16 tokens is one contiguous bulk
// copy of 32 * d bytes.
//
// Two kernels share the group step:
//   rows     16 rows per CTA; its four warps take the groups of a split in
//            turn, each with its own ring of bulk copies and its own softmax
//            state, and merge at the end.  HBM bound: every (request, head)
//            reads its codes once.  For single tokens and short chunks.
//   prompt   8 warps of 16 or 32 rows each share every group of codes; a
//            ninth warp keeps the ring full.  Bound by the tensor pipe and
//            the instructions that feed it.
// Splits of the key axis leave (m, l, O) partials that a third kernel joins
// in split order, so results do not depend on timing.
#include "kernels_kv8.hpp"

#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace kqb {

namespace {

constexpr uint32_t kG = kKv8GroupTokens;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kRaise = 8.0f;        // a logit this far above m raises it
constexpr float kWeightScale = 64.0f; // 2^6
constexpr uint32_t kWaitPolls = 1u << 22;

__device__ __forceinline__ bool err_raised(const ErrorWord &e) {
    return *reinterpret_cast<volatile unsigned long long *>(e.word) != 0ull;
}

__device__ __forceinline__ void raise(const ErrorWord &e, uint32_t code) {
    atomicCAS(e.word, 0ull, ((unsigned long long)code << 32) | e.call_id);
}

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bulk_copy(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

__device__ __forceinline__ void bar_init(uint64_t *bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}

__device__ __forceinline__ void bar_expect(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

__device__ __forceinline__ void bar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Bounded wait for the phase of `bar` with the given parity.
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity) {
    const uint32_t a = smem_u32(bar);
    for (uint32_t i = 0; i < kWaitPolls; ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.b32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(a), "r"(parity)
            : "memory");
        if (done) return true;
    }
    return false;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// What fp16 rounding of (lo, hi) left behind, as fp16.
__device__ __forceinline__ uint32_t pack_rest(float lo, float hi, uint32_t packed) {
    const __half2 h = *reinterpret_cast<const __half2 *>(&packed);
    return pack_half(lo - __low2float(h), hi - __high2float(h));
}

// Four stored bytes -> two fp16 pairs, exactly.  int8: each byte becomes the
// low mantissa bits of 1024 (one PRMT per pair), and 1024 + 128 come off.
template <bool E4M3>
__device__ __forceinline__ void widen(uint32_t w, uint32_t &b0, uint32_t &b1) {
    if constexpr (E4M3) {
        asm("{\n\t.reg .b16 x, y;\n\t"
            "mov.b32 {x, y}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, x;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, y;\n\t}"
            : "=r"(b0), "=r"(b1)
            : "r"(w));
    } else {
        const uint32_t c = 0x64646464u;
        const uint32_t x = __byte_perm(w, c, 0x4140), y = __byte_perm(w, c, 0x4342);
        const __half2 bias = __half2(__ushort_as_half(0xE480), __ushort_as_half(0xE480));   // -1152
        const __half2 u = __hadd2(*reinterpret_cast<const __half2 *>(&x), bias);
        const __half2 v = __hadd2(*reinterpret_cast<const __half2 *>(&y), bias);
        b0 = *reinterpret_cast<const uint32_t *>(&u);
        b1 = *reinterpret_cast<const uint32_t *>(&v);
    }
}

// The key/value groups that the rows of one tile can see, and where its
// request stands.
struct Request {
    uint32_t first, n, length;   // first query token, query tokens, cached tokens (new ones included)
};

// Reads and checks request b of the step; false (and an error) if its entries
// are out of range.
__device__ __forceinline__ bool load_request(const Kv8Cache &c, const Kv8Step &s, uint32_t b, Request &r,
                                             const ErrorWord &err) {
    const int32_t o0 = s.query_offsets[b], o1 = s.query_offsets[b + 1], len = s.kv_lengths[b];
    const bool ok = o0 >= 0 && o1 >= o0 && (uint32_t)o1 <= s.tokens && len >= 0 &&
                    (uint64_t)len <= (uint64_t)s.columns * c.page_tokens;
    r.first = (uint32_t)o0;
    r.n = (uint32_t)(o1 - o0);
    r.length = (uint32_t)len;
    if (!ok) raise(err, kErrStep);
    return ok;
}

// How a warp's 16 MMA rows are used:
//   kPlain    16 query rows, fp16-exact queries (bfloat16)
//   kTwoTerm  16 query rows, every product in two terms (F32)
//   kStacked  8 query rows: rows 0-7 hold the high parts of Q and of the
//             weights, rows 8-15 the low parts (F32), so that one product
//             does both; the halves meet in the same thread's registers
enum Mode { kPlain, kTwoTerm, kStacked };
constexpr int terms_of(int mode) { return mode == kTwoTerm ? 2 : 1; }
constexpr int rows_of(int mode) { return mode == kStacked ? 8 : 16; }

// One tile per warp and MT: softmax state and accumulators.  Thread (g, t) =
// (lane / 4, lane % 4) holds rows g and, except when stacked, g + 8.
template <int D, int MT>
struct Rows {
    float o[MT][D / 8][4];
    float m[MT][2], l[MT][2], ref;

    __device__ __forceinline__ void clear() {
        ref = 0.0f;
#pragma unroll
        for (int a = 0; a < MT; ++a) {
#pragma unroll
            for (int h = 0; h < 2; ++h) m[a][h] = -INFINITY, l[a][h] = 0.0f;
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[a][n][k] = 0.0f;
        }
    }
};

// One step over NG groups of 16 consecutive tokens each (`kv`: their codes in
// shared memory, 32 * D bytes a group).  q: the rows' fragments
// [MT][TERMS][D / 16][32 lanes].  factor: per row, softmax scale * log2 e /
// the row's power of two.  limit: last visible token per row (-1: none);
// compared only when MASK.
// The first product's sums run in eight independent accumulators per thread
// (CH chains per tile): a chain of D / 16 dependent MMAs per group was what
// the row kernel waited for (302 us against 225 for 64 F32 sequences).
template <int D, int MT, int NG, int MODE, bool E4M3, bool MASK>
__device__ __forceinline__ void group_step(Rows<D, MT> &st, const uint4 *q, const uint8_t *kv, const float (&ks)[NG],
                                           const float (&vs)[NG], const float (&factor)[MT][2],
                                           const int32_t (&limit)[MT][2], int32_t token, uint32_t lane) {
    constexpr int TERMS = terms_of(MODE), R = MODE == kStacked ? 1 : 2;
    constexpr int CH = MT * NG >= 4 ? 1 : 4 / (MT * NG);
    float s[MT][NG][2][4];
    {
        float c[CH][MT][NG][2][4];
#pragma unroll
        for (int x = 0; x < CH; ++x)
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int n = 0; n < NG; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int k = 0; k < 4; ++k) c[x][a][n][h][k] = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            uint4 w[NG][2];
#pragma unroll
            for (int n = 0; n < NG; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    w[n][h] = *reinterpret_cast<const uint4 *>(kv + n * 32 * D + j * 1024 + h * 512 + lane * 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t b[NG][2][2];
#pragma unroll
                for (int n = 0; n < NG; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint4 &x = w[n][h];
                        widen<E4M3>(i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w, b[n][h][0], b[n][h][1]);
                    }
#pragma unroll
                for (int a = 0; a < MT; ++a)
#pragma unroll
                    for (int term = TERMS - 1; term >= 0; --term) {
                        const uint4 f = q[((a * TERMS + term) * (D / 16) + j * 4 + i) * 32 + lane];
#pragma unroll
                        for (int n = 0; n < NG; ++n)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                mma(c[(i * TERMS + term) % CH][a][n][h], f, b[n][h][0], b[n][h][1]);
                    }
            }
        }
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int n = 0; n < NG; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float v = c[0][a][n][h][k];
#pragma unroll
                        for (int x = 1; x < CH; ++x) v += c[x][a][n][h][k];
                        s[a][n][h][k] = v;
                    }
    }

    // logits, the rows' maxima
    float top[MT][R];
    bool lift = false;
#pragma unroll
    for (int a = 0; a < MT; ++a) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float x = -INFINITY;
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                const float f = factor[a][r] * ks[n];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float v = s[a][n][h][2 * r + k];
                        if constexpr (MODE == kStacked) v += s[a][n][h][2 + k];
                        v *= f;
                        if (MASK && token + n * 16 + h * 8 + (int32_t)(lane & 3) * 2 + k > limit[a][r]) v = -INFINITY;
                        s[a][n][h][2 * r + k] = v;
                        x = fmaxf(x, v);
                    }
            }
            x = fmaxf(x, __shfl_xor_sync(~0u, x, 1));
            x = fmaxf(x, __shfl_xor_sync(~0u, x, 2));
            top[a][r] = x;
            lift |= x > st.m[a][r] + kRaise;
        }
    }
    if (__any_sync(~0u, lift)) {   // -inf + 8 is -inf: the first finite logit of a row lifts it
#pragma unroll
        for (int a = 0; a < MT; ++a) {
            float by[2];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float m = fmaxf(st.m[a][r], top[a][r]);
                by[r] = m == -INFINITY ? 1.0f : exp2_approx(st.m[a][r] - m);
                st.m[a][r] = m;
                st.l[a][r] *= by[r];
            }
            if constexpr (R == 1) by[1] = by[0];
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) st.o[a][n][k] *= by[k >> 1];
        }
    }
    float most = vs[0];
#pragma unroll
    for (int n = 1; n < NG; ++n) most = fmaxf(most, vs[n]);
    if (most > st.ref) {
        // the next power of two, within the normal range
        const uint32_t e = min((__float_as_uint(most) + 0x7fffffu) & 0x7f800000u, 0x7f000000u);
        const float ref = __uint_as_float(max(e, 0x00800000u));
        const float by = st.ref / ref;
        st.ref = ref;
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) st.o[a][n][k] *= by;
    }
    const float inv = st.ref > 0.0f ? kWeightScale / st.ref : 0.0f;

    // weights, as the second product's A operand
    uint4 p[MT][NG][TERMS];
#pragma unroll
    for (int a = 0; a < MT; ++a) {
        float m[2];
#pragma unroll
        for (int r = 0; r < R; ++r) m[r] = st.m[a][r] == -INFINITY ? 0.0f : st.m[a][r];
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            const float w = vs[n] * inv;
            float e[2][2 * R];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int k = 0; k < 2 * R; ++k) {
                    e[h][k] = exp2_approx(s[a][n][h][k] - m[k >> 1]);
                    st.l[a][k >> 1] += e[h][k];
                    e[h][k] *= w;
                }
            }
            if constexpr (MODE == kStacked) {
                const uint32_t h0 = pack_half(e[0][0], e[0][1]), h1 = pack_half(e[1][0], e[1][1]);
                p[a][n][0] = make_uint4(h0, pack_rest(e[0][0], e[0][1], h0), h1, pack_rest(e[1][0], e[1][1], h1));
            } else {
                p[a][n][0] = make_uint4(pack_half(e[0][0], e[0][1]), pack_half(e[0][2], e[0][3]),
                                        pack_half(e[1][0], e[1][1]), pack_half(e[1][2], e[1][3]));
                if constexpr (TERMS == 2)
                    p[a][n][1] =
                        make_uint4(pack_rest(e[0][0], e[0][1], p[a][n][0].x), pack_rest(e[0][2], e[0][3], p[a][n][0].y),
                                   pack_rest(e[1][0], e[1][1], p[a][n][0].z), pack_rest(e[1][2], e[1][3], p[a][n][0].w));
            }
        }
    }

#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
        uint4 w[NG];
#pragma unroll
        for (int n = 0; n < NG; ++n)
            w[n] = *reinterpret_cast<const uint4 *>(kv + n * 32 * D + 16 * D + j * 512 + lane * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t b[NG][2];
#pragma unroll
            for (int n = 0; n < NG; ++n)
                widen<E4M3>(i == 0 ? w[n].x : i == 1 ? w[n].y : i == 2 ? w[n].z : w[n].w, b[n][0], b[n][1]);
#pragma unroll
            for (int a = 0; a < MT; ++a) {
                if constexpr (TERMS == 2) {
                    // a fresh accumulator per step, added in F32: the tensor
                    // core's own addition truncates, and over thousands of
                    // groups that bias would exceed F32's rounding
                    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int n = 0; n < NG; ++n) {
                        mma(d, p[a][n][1], b[n][0], b[n][1]);
                        mma(d, p[a][n][0], b[n][0], b[n][1]);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) st.o[a][j * 4 + i][k] += d[k];
                } else {
#pragma unroll
                    for (int n = 0; n < NG; ++n) mma(st.o[a][j * 4 + i], p[a][n][0], b[n][0], b[n][1]);
                }
            }
        }
    }
}

// Writes rows [row0, row0 + rows_in_tile) of request `rq` as fragments into q
// and, per row, 1 / its power of two (times the softmax scale in base 2) into
// factor and its last visible token into limit.  Eight threads per row, every
// thread of the CTA takes part; rows behind the request's last are zero with
// limit -1.  Returns whether a query value was not finite.
template <int D, int MODE, int THREADS, int ROWS>
__device__ __forceinline__ bool load_queries(const Kv8Attend &a, const Request &rq, uint32_t G, uint32_t head,
                                             uint32_t row0, uint4 *q, float *factor, int32_t *limit, uint32_t tid) {
    constexpr int TERMS = terms_of(MODE);
    bool bad = false;
    uint32_t *q32 = reinterpret_cast<uint32_t *>(q);
    const uint32_t part = tid & 7;
    for (uint32_t r = tid >> 3; r < ROWS; r += THREADS / 8) {
        const uint32_t row = row0 + r, token = row / G;
        const bool live = token < rq.n;
        float x[D / 8];
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (live) {
                const uint64_t at = (uint64_t)(rq.first + token) * a.q_stride + (uint64_t)(head * G + row % G) * D +
                                    (part + 8 * k) * 4;
                if constexpr (MODE == kPlain) {
                    const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const __nv_bfloat16 *>(a.q) + at);
                    v = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u),
                                    __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
                } else {
                    v = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + at);
                }
            }
            x[4 * k] = v.x, x[4 * k + 1] = v.y, x[4 * k + 2] = v.z, x[4 * k + 3] = v.w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bad |= !(fabsf(x[4 * k + i]) < INFINITY);
                top = fmaxf(top, fabsf(x[4 * k + i]));
            }
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        // the row's largest element into [2^13, 2^14); 2^-100 is the smallest that is still scaled
        const int e = max((int)(__float_as_uint(top) >> 23), 27) - 127 - 13;
        const float up = __uint_as_float((uint32_t)(127 - e) << 23), down = __uint_as_float((uint32_t)(127 + e) << 23);
        const uint32_t tile = r >> 4, half = r >> 3 & 1;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            const uint32_t f = (part + 8 * k) * 4;
            const uint32_t at = (((tile * TERMS) * (D / 16) + f / 64 * 4 + f % 16 / 4) * 32 + (r & 7) * 4 + f % 64 / 16) * 4 + half;
            const uint32_t h0 = pack_half(x[4 * k] * up, x[4 * k + 1] * up), h1 = pack_half(x[4 * k + 2] * up, x[4 * k + 3] * up);
            q32[at] = h0;
            q32[at + 2] = h1;
            if constexpr (MODE != kPlain) {
                constexpr uint32_t low = MODE == kStacked ? 1 : D / 16 * 128;   // rows 8-15, or the second term
                q32[at + low] = pack_rest(x[4 * k] * up, x[4 * k + 1] * up, h0);
                q32[at + low + 2] = pack_rest(x[4 * k + 2] * up, x[4 * k + 3] * up, h1);
            }
        }
        if (part == 0) {
            factor[r] = a.scale_log2 * down;
            limit[r] = live ? (int32_t)(rq.length - rq.n + token) : -1;
        }
    }
    return bad;
}

// A finished row's value and its log-sum, or a split's partial.
template <bool BF16>
__device__ __forceinline__ void store4(void *out, uint64_t at, float4 v) {
    if constexpr (BF16) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(v.x, v.y), y = __floats2bfloat162_rn(v.z, v.w);
        *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(out) + at) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
    } else {
        *reinterpret_cast<float4 *>(static_cast<float *>(out) + at) = v;
    }
}

// Where the partials of a (tile, head) lie: O [split][row][D], and behind the
// O of all `tiles`, (m, l) [row][split].
struct Partials {
    float *o;
    float2 *ml;
    __device__ __forceinline__ Partials(float *base, uint64_t tile, uint32_t splits, uint32_t rows, uint32_t dim,
                                        uint64_t tiles) {
        o = base + tile * splits * rows * dim;
        ml = reinterpret_cast<float2 *>(base + tiles * splits * rows * dim) + tile * rows * splits;
    }
};

// Groups of 16 tokens that the rows up to `last_row` of a request see.
__device__ __forceinline__ uint32_t visible_groups(const Request &rq, uint32_t G, uint32_t rows_end) {
    const uint32_t token = (rows_end - 1) / G;   // the tile's last token
    const int64_t last = (int64_t)rq.length - rq.n + min(token, rq.n - 1);
    return last < 0 ? 0u : (uint32_t)(last / kG) + 1u;
}

// A split's groups: at least `each`, never more splits than the launch has,
// and whole stages (`unit` groups, which `each` is a multiple of).
__device__ __forceinline__ uint32_t split_groups(uint32_t groups, uint32_t each, uint32_t splits, uint32_t unit) {
    return max(each, ((groups + splits - 1) / splits + unit - 1) / unit * unit);
}

template <int D> constexpr int kRowStages = D == 256 ? 3 : 6;
constexpr int kRowWarps = 4;
template <int D, int TERMS> constexpr uint32_t kRowSmem = kRowWarps * kRowStages<D> * 32 * D + TERMS * 32 * D;

}  // namespace

// grid (request, tile, head, split); four warps, 16 or 8 rows.  Each warp streams
// every fourth group of the split through its own ring; page ids and scales of
// a warp's next 32 groups sit in its lanes.
// Partials: [request][tile][head][split][16 rows][D], then (m, l) per row.
template <int D, int MODE, bool E4M3>
__global__ void __launch_bounds__(kRowWarps * 32, 2)
kv8_rows_kernel(Kv8Cache c, Kv8Step s, Kv8Attend a, Kv8Shape shape, ErrorWord err) {
    constexpr int ST = kRowStages<D>;
    constexpr bool BF16 = MODE == kPlain;
    constexpr uint32_t kStage = 32 * D, kRows = rows_of(MODE), kR = MODE == kStacked ? 1 : 2;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[kRowWarps][ST];
    __shared__ float factor_s[16], merge_m[kRowWarps][16], merge_l[kRowWarps][16];
    __shared__ int32_t limit_s[16];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint8_t *ring = smem + warp * ST * kStage;
    uint4 *q = reinterpret_cast<uint4 *>(smem + kRowWarps * ST * kStage);
    const uint32_t G = a.query_heads / c.heads;
    const uint32_t split = blockIdx.x % shape.row_splits, u = blockIdx.x / shape.row_splits;
    const uint32_t head = u % c.heads, tile0 = u / c.heads % shape.row_tiles, b = u / c.heads / shape.row_tiles;

    if (tid < kRowWarps * ST) bar_init(&full[0][0] + tid, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    pdl_wait();
    if (__syncthreads_or(tid == 0 && err_raised(err))) return;
    Request rq;
    if (!load_request(c, s, b, rq, err)) return;
    const uint64_t rows64 = (uint64_t)rq.n * G;
    if (rows64 == 0 || rows64 > shape.row_limit) return;
    const uint32_t rows = (uint32_t)rows64;
    // a request of more tiles than the launch has is not split: its partials
    // would have no place
    const uint32_t splits = (rows + kRows - 1) / kRows > shape.row_tiles ? 1u : shape.row_splits;
    const int32_t *table = s.table + (uint64_t)b * s.table_stride;
    const uint32_t per_page = c.page_tokens / kG;
    const uint64_t page_bytes = 2ull * c.page_tokens * D;
    uint32_t used = 0;   // ring slots used so far (waits go by it)

    for (uint32_t tile = tile0; tile * kRows < rows; tile += shape.row_tiles) {
        const uint32_t row0 = tile * kRows, row_end = min(row0 + kRows, rows);
        const uint32_t groups = visible_groups(rq, G, row_end), each = split_groups(groups, shape.row_groups, splits, 1);
        const uint32_t g0 = split * each, g1 = min(g0 + each, groups);
        if (split > 0 && g0 >= groups) break;   // later tiles see more groups only when splits == 1
        // this warp's groups: g0 + warp + 4 i
        const uint32_t mine = g1 > g0 + warp ? (g1 - g0 - warp + kRowWarps - 1) / kRowWarps : 0;
        uint32_t page = 0;
        float2 scales = make_float2(0.0f, 0.0f);
        auto fetch = [&](uint32_t from) {   // page ids and scales of groups from .. from + 31
            const uint32_t i = from + lane;
            if (i < mine) {
                const int32_t id = table[(g0 + warp + i * kRowWarps) / per_page];
                const bool ok = id >= 0 && (uint32_t)id < c.pages;
                if (!ok) raise(err, kErrStep);
                page = ok ? (uint32_t)id : 0u;   // any page: the call fails
                scales = *reinterpret_cast<const float2 *>(c.scales + ((uint64_t)page * c.heads + head) * 2);
            }
        };
        auto issue = [&](uint32_t i) {   // group i of this warp into its slot; page ids are in the lanes
            const uint32_t id = __shfl_sync(~0u, page, i & 31);
            if (lane == 0) {
                const uint32_t slot = (used + i) % ST;
                bar_expect(&full[warp][slot], kStage);
                bulk_copy(ring + slot * kStage,
                          c.codes + ((uint64_t)id * c.heads + head) * page_bytes +
                              (uint64_t)((g0 + warp + i * kRowWarps) % per_page) * kStage,
                          kStage, &full[warp][slot]);
            }
        };
        fetch(0);
        uint32_t issued = 0;
        for (; issued < min(mine, (uint32_t)ST); ++issued) issue(issued);

        if (load_queries<D, MODE, kRowWarps * 32, kRows>(a, rq, G, head, row0, q, factor_s, limit_s, tid))
            raise(err, kErrNonFinite);
        __syncthreads();
        Rows<D, 1> st;
        st.clear();
        const float factor[1][2] = {{factor_s[lane >> 2], factor_s[(lane >> 2) + 8 * (kR - 1)]}};
        const int32_t limit[1][2] = {{limit_s[lane >> 2], limit_s[(lane >> 2) + 8 * (kR - 1)]}};
        // every row of the tile sees the tokens up to its first token's
        const uint32_t clear_to = rq.length + 1 > rq.n ? rq.length - rq.n + row0 / G + 1 : 0u;
        bool ok = true;
        uint32_t i = 0;
        for (; i < mine && ok; ++i) {
            if (i > 0 && (i & 31) == 0) {
                // the lanes' next 32 groups; the ring runs dry here once per 128 groups of the split
                fetch(i);
                for (; issued < min(mine, i + ST); ++issued) issue(issued);
            }
            const uint32_t slot = (used + i) % ST;
            ok = bar_wait(&full[warp][slot], (used + i) / ST & 1u);
            if (!ok) break;
            const float ks[1] = {__shfl_sync(~0u, scales.x, i & 31)}, vs[1] = {__shfl_sync(~0u, scales.y, i & 31)};
            const uint32_t token = (g0 + warp + i * kRowWarps) * kG;
            const uint8_t *kv = ring + slot * kStage;
            if (token + kG > clear_to || row_end < row0 + kRows)
                group_step<D, 1, 1, MODE, E4M3, true>(st, q, kv, ks, vs, factor, limit, (int32_t)token, lane);
            else
                group_step<D, 1, 1, MODE, E4M3, false>(st, q, kv, ks, vs, factor, limit, (int32_t)token, lane);
            __syncwarp();
            // refill only with groups whose page ids the lanes hold
            if (issued < mine && (issued & ~31u) == (i & ~31u)) issue(issued++);
        }
        if (!ok) {
            // a wait gave up: let the other copies land before the CTA exits
            if (lane == 0) raise(err, kErrTimeout);
            for (uint32_t k = i; k < issued; ++k) bar_wait(&full[warp][(used + k) % ST], (used + k) / ST & 1u);
        }
        used += mine;

        // join the warps: (m, l) and O of each in its own ring
#pragma unroll
        for (int r = 0; r < (int)kR; ++r) {
            st.l[0][r] += __shfl_xor_sync(~0u, st.l[0][r], 1);
            st.l[0][r] += __shfl_xor_sync(~0u, st.l[0][r], 2);
        }
        if ((lane & 3) == 0) {
#pragma unroll
            for (int r = 0; r < (int)kR; ++r) {
                merge_m[warp][(lane >> 2) + 8 * r] = st.m[0][r];
                merge_l[warp][(lane >> 2) + 8 * r] = st.l[0][r];
            }
        }
        constexpr uint32_t kPitch = D + 4;   // rows 4 banks apart: conflict-free 16-byte stores
        float *mo = reinterpret_cast<float *>(ring);
        const float back = st.ref * (1.0f / kWeightScale);
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int r = 0; r < (int)kR; ++r)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[i] = st.o[0][4 * j + i][2 * r + k];
                        if constexpr (MODE == kStacked) x[i] += st.o[0][4 * j + i][2 + k];
                        x[i] *= back;
                    }
                    *reinterpret_cast<float4 *>(mo + ((lane >> 2) + 8 * r) * kPitch + j * 32 + (lane & 3) * 8 + 4 * k) =
                        make_float4(x[0], x[1], x[2], x[3]);
                }
        __syncthreads();
        const bool whole = groups <= each;   // one split: the result itself
        const Partials part(a.workspace, ((uint64_t)b * shape.row_tiles + tile) * c.heads + head, shape.row_splits, 16, D,
                            (uint64_t)s.requests * shape.row_tiles * c.heads);
        for (uint32_t v = tid; v < (row_end - row0) * (D / 4); v += kRowWarps * 32) {
            const uint32_t r = v / (D / 4), f = v % (D / 4) * 4;
            float m = merge_m[0][r];
#pragma unroll
            for (int w = 1; w < kRowWarps; ++w) m = fmaxf(m, merge_m[w][r]);
            float l = 0.0f;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) {
                const float by = merge_m[w][r] == -INFINITY ? 0.0f : exp2_approx(merge_m[w][r] - m);
                const float4 x = *reinterpret_cast<const float4 *>(
                    reinterpret_cast<const float *>(smem + w * ST * kStage) + r * kPitch + f);
                l += merge_l[w][r] * by;
                o.x += x.x * by, o.y += x.y * by, o.z += x.z * by, o.w += x.w * by;
            }
            if (whole) {
                const float inv = l > 0.0f ? 1.0f / l : 0.0f;
                o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
                if (!(l < INFINITY) || !(fabsf(o.x) + fabsf(o.y) + fabsf(o.z) + fabsf(o.w) < INFINITY))
                    raise(err, kErrNonFinite);
                const uint32_t row = row0 + r, token = rq.first + row / G, qh = head * G + row % G;
                store4<BF16>(a.out, (uint64_t)token * a.out_stride + (uint64_t)qh * D + f, o);
                if (a.lse != nullptr && f == 0)
                    a.lse[(uint64_t)token * a.query_heads + qh] = l > 0.0f ? (m + log2f(l)) * kLn2 : -INFINITY;
            } else {
                *reinterpret_cast<float4 *>(part.o + ((uint64_t)split * 16 + r) * D + f) = o;
                if (f == 0) part.ml[r * shape.row_splits + split] = make_float2(m, l);
            }
        }
        if (__syncthreads_or(!ok)) return;
        // the ring, the queries and the merge are free again; the ring's next
        // writes come through the asynchronous proxy
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
}

namespace {

// ----------------------------------------------------------------- prompt

constexpr int kPromptWarps = 8;
constexpr int kPromptThreads = (kPromptWarps + 4) * 32;
constexpr int kPromptGroups = 2;   // groups per ring stage
template <int D> constexpr int kPromptMt = D == 256 ? 1 : 2;
template <int D> constexpr uint32_t kPromptRows = kPromptWarps * 16 * kPromptMt<D>;
template <int D> constexpr int kPromptStages = D == 256 ? 4 : 8;
template <int D, int TERMS>
constexpr uint32_t kPromptSmem = kPromptStages<D> * kPromptGroups * 32 * D + kPromptRows<D> * D * 2 * TERMS;

// The request and tile of compact tile index t: request b's tiles begin at
// floor(offset_b * G / rows) + b, which leaves room for its partial tile.
// The warp searches 32 ways at a time.
__device__ __forceinline__ uint32_t find_request(const Kv8Step &s, uint32_t G, uint32_t tile_rows, uint32_t t,
                                                 uint32_t lane, uint32_t &start) {
    uint32_t lo = 0, n = s.requests;   // the answer lies in [lo, lo + n)
    auto begin = [&](uint32_t b) {
        return (uint32_t)((uint64_t)(uint32_t)max(s.query_offsets[b], 0) * G / tile_rows) + b;
    };
    while (n > 1) {
        const uint32_t step = (n + 31) / 32, at = lo + lane * step;
        const bool in = lane * step < n && begin(at) <= t;
        const uint32_t hits = __ballot_sync(~0u, in);
        const uint32_t k = hits ? 31 - __clz(hits) : 0u;
        const uint32_t end = lo + n;
        lo += k * step;
        n = min(step, end - lo);
    }
    start = begin(lo);
    return lo;
}

}  // namespace

// grid (tile, head, split), the last tiles first (they see the most tokens).
// Warp w < 8 holds rows [16 MT w, 16 MT (w + 1)) of the tile; warp 8 streams
// the split's groups, two to a stage, and leaves their scales beside them.
// Registers: 384 threads of 168 at launch (64,512); the consumers' two
// warpgroups take 232 each thread, the producer's keeps 40 (the same sum).
template <int D, bool BF16, bool E4M3>
__global__ void __launch_bounds__(kPromptThreads, 1)
kv8_prompt_kernel(Kv8Cache c, Kv8Step s, Kv8Attend a, Kv8Shape shape, ErrorWord err) {
    constexpr int MODE = BF16 ? kPlain : kTwoTerm, TERMS = terms_of(MODE), MT = kPromptMt<D>, ST = kPromptStages<D>, NG = kPromptGroups;
    constexpr uint32_t kGroup = 32 * D, kStage = NG * kGroup, kRows = kPromptRows<D>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[ST], empty[ST];
    __shared__ float2 stage_scales[ST][NG];
    __shared__ float factor_s[kRows];
    __shared__ int32_t limit_s[kRows];
    __shared__ int gave_up;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint4 *q = reinterpret_cast<uint4 *>(smem + ST * kStage);
    const uint32_t G = a.query_heads / c.heads;
    const uint32_t split = blockIdx.x % shape.prompt_splits, u = blockIdx.x / shape.prompt_splits;
    const uint32_t head = u % c.heads, t = shape.prompt_tiles - 1 - u / c.heads;

    if (tid == 0) {
        gave_up = 0;
        for (int k = 0; k < ST; ++k) {
            bar_init(&full[k], NG);
            bar_init(&empty[k], kPromptWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    if (__syncthreads_or(tid == 0 && err_raised(err))) return;
    uint32_t start;
    const uint32_t b = find_request(s, G, kRows, t, lane, start);
    Request rq;
    if (!load_request(c, s, b, rq, err)) return;
    const uint64_t rows64 = (uint64_t)rq.n * G;
    if (t < start || rows64 <= shape.row_limit || (uint64_t)(t - start) * kRows >= rows64) return;
    const uint32_t rows = (uint32_t)rows64, row0 = (t - start) * kRows, row_end = min(row0 + kRows, rows);
    const uint32_t groups = visible_groups(rq, G, row_end), each = split_groups(groups, shape.prompt_groups, shape.prompt_splits, NG);
    const uint32_t g0 = split * each, g1 = min(g0 + each, groups);
    if (split > 0 && g0 >= groups) return;
    const uint32_t stages = g1 > g0 ? (g1 - g0 + NG - 1) / NG : 0u;
    volatile int *quit = &gave_up;

    if (warp >= kPromptWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        // producer: lane k < NG of warp 8 brings group k of every stage (behind
        // an odd last group that group again: its tokens are behind every
        // row's limit then)
        bool ok = true;
        uint32_t done = 0;
        if (warp == kPromptWarps && lane < NG) {
            const int32_t *table = s.table + (uint64_t)b * s.table_stride;
            const uint32_t per_page = c.page_tokens / kG;
            const uint64_t page_bytes = 2ull * c.page_tokens * D;
            int32_t next = stages > 0 ? table[min(g0 + lane, g1 - 1) / per_page] : 0;
            for (uint32_t k = 0; k < stages && !*quit; ++k) {
                const uint32_t slot = k % ST, g = min(g0 + k * NG + lane, g1 - 1);
                const bool in = next >= 0 && (uint32_t)next < c.pages;
                if (!in) raise(err, kErrStep);
                const uint32_t page = in ? (uint32_t)next : 0u;   // any page: the call fails
                if (k + 1 < stages) next = table[min(g + NG, g1 - 1) / per_page];
                const float2 sc = *reinterpret_cast<const float2 *>(c.scales + ((uint64_t)page * c.heads + head) * 2);
                if (k >= ST) ok = bar_wait(&empty[slot], (k / ST - 1) & 1u);
                if (!ok) break;
                stage_scales[slot][lane] = sc;
                bar_expect(&full[slot], kGroup);
                bulk_copy(smem + slot * kStage + lane * kGroup,
                          c.codes + ((uint64_t)page * c.heads + head) * page_bytes + (uint64_t)(g % per_page) * kGroup,
                          kGroup, &full[slot]);
                done = k + 1;
            }
            if (!ok) {
                raise(err, kErrTimeout);
                *quit = 1;
            }
        }
        __syncwarp();
        asm volatile("bar.sync 0;" ::: "memory");
        if (warp == kPromptWarps && lane < NG && *quit)   // copies in flight land before the CTA exits
            for (uint32_t k = done > ST ? done - ST : 0u; k < done; ++k) bar_wait(&full[k % ST], k / ST & 1u);
        return;
    }
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");

    if (load_queries<D, MODE, kPromptWarps * 32, kRows>(a, rq, G, head, row0, q, factor_s, limit_s, tid))
        raise(err, kErrNonFinite);
    asm volatile("bar.sync 1, %0;" ::"n"(kPromptWarps * 32) : "memory");
    Rows<D, MT> st;
    st.clear();
    float factor[MT][2];
    int32_t limit[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint32_t row = (warp * MT + m) * 16 + (lane >> 2) + 8 * r;
            factor[m][r] = factor_s[row];
            limit[m][r] = limit_s[row];
        }
    // tokens that every row of the warp sees, and that any does
    const uint32_t first_row = row0 + warp * MT * 16;
    const int64_t before = (int64_t)rq.length - rq.n;
    const bool warp_live = first_row < row_end;
    const int64_t all_see = warp_live && first_row + MT * 16 <= row_end ? before + first_row / G + 1 : 0;
    const int64_t any_sees = warp_live ? before + (min(first_row + MT * 16, row_end) - 1) / G + 1 : 0;
    const uint4 *wq = q + warp * MT * TERMS * (D / 16) * 32;
    bool ok = true;
    for (uint32_t k = 0; k < stages; ++k) {
        const uint32_t slot = k % ST;
        ok = !*quit && bar_wait(&full[slot], k / ST & 1u);
        if (!ok) break;
        const int64_t token = (int64_t)(g0 + k * NG) * kG;
        if (token < any_sees) {
            const float2 s0 = stage_scales[slot][0], s1 = stage_scales[slot][1];
            const float ks[NG] = {s0.x, s1.x}, vs[NG] = {s0.y, s1.y};
            const uint8_t *kv = smem + slot * kStage;
            if (token + NG * kG > all_see || g0 + (k + 1) * NG > g1)
                group_step<D, MT, NG, MODE, E4M3, true>(st, wq, kv, ks, vs, factor, limit, (int32_t)token, lane);
            else
                group_step<D, MT, NG, MODE, E4M3, false>(st, wq, kv, ks, vs, factor, limit, (int32_t)token, lane);
        }
        __syncwarp();
        if (lane == 0) bar_arrive(&empty[slot]);
    }
    if (!ok) {
        if (lane == 0) {
            *quit = 1;
            raise(err, kErrTimeout);
        }
    }
    asm volatile("bar.sync 0;" ::: "memory");
    if (!ok) return;

    const bool whole = groups <= each;
    const Partials part(a.workspace + shape.row_floats, (uint64_t)t * c.heads + head, shape.prompt_splits, kRows, D,
                        (uint64_t)shape.prompt_tiles * c.heads);
    const float back = st.ref * (1.0f / kWeightScale);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float l = st.l[m][r];
            l += __shfl_xor_sync(~0u, l, 1);
            l += __shfl_xor_sync(~0u, l, 2);
            const uint32_t in_tile = (warp * MT + m) * 16 + (lane >> 2) + 8 * r, row = row0 + in_tile;
            if (row >= row_end) continue;
            const uint32_t token = rq.first + row / G, qh = head * G + row % G;
            const float by = whole ? (l > 0.0f ? back / l : 0.0f) : back;
            bool fine = l < INFINITY;
#pragma unroll
            for (int j = 0; j < D / 32; ++j)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float4 o = make_float4(st.o[m][4 * j][2 * r + k] * by, st.o[m][4 * j + 1][2 * r + k] * by,
                                                 st.o[m][4 * j + 2][2 * r + k] * by, st.o[m][4 * j + 3][2 * r + k] * by);
                    const uint32_t f = j * 32 + (lane & 3) * 8 + 4 * k;
                    if (whole) {
                        fine &= fabsf(o.x) + fabsf(o.y) + fabsf(o.z) + fabsf(o.w) < INFINITY;
                        store4<BF16>(a.out, (uint64_t)token * a.out_stride + (uint64_t)qh * D + f, o);
                    } else {
                        *reinterpret_cast<float4 *>(part.o + ((uint64_t)split * kRows + in_tile) * D + f) = o;
                    }
                }
            if ((lane & 3) == 0) {
                if (!whole)
                    part.ml[in_tile * shape.prompt_splits + split] = make_float2(st.m[m][r], l);
                else if (a.lse != nullptr)
                    a.lse[(uint64_t)token * a.query_heads + qh] = l > 0.0f ? (st.m[m][r] + log2f(l)) * kLn2 : -INFINITY;
            }
            if (whole && !fine) raise(err, kErrNonFinite);
        }
}

constexpr int kJoinThreads = 256;

// Joins the splits of a row: one CTA per (tile, head, row), or per 64 features
// of it where there are few.  The threads first turn the splits' (m, l) into
// weights 2^(m_k - m) in shared memory, 1024 at a time; 16 threads then hold 4
// features each of every 16th split, and meet in shared memory in a fixed
// order.  Bound: latency, the partials come from L2.
template <int D, bool BF16>
__global__ void __launch_bounds__(kJoinThreads)
kv8_join_kernel(Kv8Cache c, Kv8Step s, Kv8Attend a, Kv8Shape shape, uint32_t prompt, ErrorWord err) {
    constexpr uint32_t kLanes = 16, kWays = kJoinThreads / kLanes, kBatch = 1024, kAhead = 8;
    __shared__ float weight[kBatch];
    __shared__ float warp_red[kJoinThreads / 32];
    __shared__ float4 way_sum[kWays][kLanes];
    const uint32_t tid = threadIdx.x, lane = tid & 31, G = a.query_heads / c.heads;
    const uint32_t tile_rows = prompt ? shape.prompt_rows : shape.join_rows;
    const uint32_t chunks = prompt ? 1u : shape.join_chunks;
    const uint32_t chunk = blockIdx.x % chunks, r0 = blockIdx.x / chunks % tile_rows;
    const uint32_t u = blockIdx.x / chunks / tile_rows, head = u % c.heads, slot = u / c.heads;
    pdl_wait();
    if (__syncthreads_or(tid == 0 && err_raised(err))) return;
    uint32_t b, tile;
    if (prompt) {
        uint32_t start;
        b = find_request(s, G, tile_rows, slot, lane, start);
        if (slot < start) return;
        tile = slot - start;
    } else {
        b = slot / shape.row_tiles;
        tile = slot % shape.row_tiles;
    }
    Request rq;
    if (!load_request(c, s, b, rq, err)) return;
    const uint64_t rows64 = (uint64_t)rq.n * G;
    const uint32_t held = prompt ? shape.prompt_rows : shape.row_tile, pitch_rows = prompt ? shape.prompt_rows : 16u;
    if (prompt ? rows64 <= shape.row_limit : rows64 > shape.row_limit) return;
    if (!prompt && (rows64 + held - 1) / held > shape.row_tiles) return;
    if ((uint64_t)tile * held >= rows64) return;
    const uint32_t rows = (uint32_t)rows64, row0 = tile * held, row_end = min(row0 + held, rows);
    const uint32_t launched = prompt ? shape.prompt_splits : shape.row_splits;
    const uint32_t groups = visible_groups(rq, G, row_end);
    const uint32_t each = split_groups(groups, prompt ? shape.prompt_groups : shape.row_groups, launched,
                                       prompt ? kPromptGroups : 1u);
    if (groups <= each) return;
    const uint32_t n = (groups + each - 1) / each;
    const Partials part(a.workspace + (prompt ? shape.row_floats : 0), (uint64_t)slot * c.heads + head, launched, pitch_rows,
                        D, (uint64_t)(prompt ? shape.prompt_tiles : s.requests * shape.row_tiles) * c.heads);

    auto all = [&](float v, bool take_max) {   // over the CTA, the same in every thread
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float x = __shfl_xor_sync(~0u, v, o);
            v = take_max ? fmaxf(v, x) : v + x;
        }
        __syncthreads();
        if (lane == 0) warp_red[tid >> 5] = v;
        __syncthreads();
        v = warp_red[0];
#pragma unroll
        for (int w = 1; w < kJoinThreads / 32; ++w) v = take_max ? fmaxf(v, warp_red[w]) : v + warp_red[w];
        return v;
    };
    const uint32_t way = tid / kLanes;
    const uint64_t pitch = (uint64_t)pitch_rows * D;
    // one row per CTA unless the tile has more than the launch expected
    for (uint32_t r = r0; row0 + r < row_end; r += tile_rows) {
        const float2 *ml = part.ml + (uint64_t)r * launched;
        float m = -INFINITY;
        for (uint32_t k = tid; k < n; k += kJoinThreads) m = fmaxf(m, ml[k].x);
        m = all(m, true);
        const uint32_t row = row0 + r, token = rq.first + row / G, qh = head * G + row % G;
        for (uint32_t f0 = chunk * 64; f0 < D; f0 += chunks * 64) {
            const uint32_t f = f0 + tid % kLanes * 4;
            const float *po = part.o + (uint64_t)r * D + f;
            float l = 0.0f;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (uint32_t k0 = 0; k0 < n; k0 += kBatch) {
                const uint32_t count = min(n - k0, kBatch);
                __syncthreads();
                for (uint32_t k = tid; k < count; k += kJoinThreads) {
                    const float2 x = ml[k0 + k];
                    const float w = x.x == -INFINITY ? 0.0f : exp2_approx(x.x - m);
                    weight[k] = w;
                    l += x.y * w;
                }
                __syncthreads();
                for (uint32_t k = way; k < count; k += kWays * kAhead) {
                    float4 y[kAhead];
#pragma unroll
                    for (uint32_t i = 0; i < kAhead; ++i)
                        y[i] = k + i * kWays < count ? *reinterpret_cast<const float4 *>(po + (k0 + k + i * kWays) * pitch)
                                                     : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (uint32_t i = 0; i < kAhead; ++i) {
                        const float w = k + i * kWays < count ? weight[k + i * kWays] : 0.0f;
                        o.x += y[i].x * w, o.y += y[i].y * w, o.z += y[i].z * w, o.w += y[i].w * w;
                    }
                }
            }
            l = all(l, false);
            way_sum[way][tid % kLanes] = o;
            __syncthreads();
            if (way == 0) {
#pragma unroll
                for (uint32_t w = 1; w < kWays; ++w) {
                    const float4 y = way_sum[w][tid];
                    o.x += y.x, o.y += y.y, o.z += y.z, o.w += y.w;
                }
                const float inv = l > 0.0f ? 1.0f / l : 0.0f;
                o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
                if (!(l < INFINITY) || !(fabsf(o.x) + fabsf(o.y) + fabsf(o.z) + fabsf(o.w) < INFINITY))
                    raise(err, kErrNonFinite);
                store4<BF16>(a.out, (uint64_t)token * a.out_stride + (uint64_t)qh * D + f, o);
                if (a.lse != nullptr && f == 0)
                    a.lse[(uint64_t)token * a.query_heads + qh] = l > 0.0f ? (m + log2f(l)) * kLn2 : -INFINITY;
            }
        }
    }
}

// --------------------------------------------------------------- launching

namespace {

constexpr uint32_t kSms = 148;
constexpr uint32_t kShortRows = 64;        // requests up to this many rows go to the row kernel
constexpr uint32_t kMaxRowGroups = 128;    // 32 groups to a warp: one batch of page ids
constexpr uint32_t kMinRowGroups = 8;
constexpr uint32_t kMinPromptGroups = 64;

template <int D, int MODE, bool E4M3>
void launch_rows(const Kv8Cache &c, const Kv8Step &s, const Kv8Attend &a, const Kv8Shape &h, ErrorWord err,
                 cudaStream_t stream) {
    static DeviceOnce once;
    once.run([] {
        cudaFuncSetAttribute(kv8_rows_kernel<D, MODE, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kRowSmem<D, terms_of(MODE)>);
    });
    KernelTimer timer("kv8_rows", stream);
    launch_pdl(kv8_rows_kernel<D, MODE, E4M3>, s.requests * h.row_tiles * c.heads * h.row_splits, kRowWarps * 32,
               kRowSmem<D, terms_of(MODE)>, stream, c, s, a, h, err);
    count_launch();
}

template <int D, bool BF16, bool E4M3>
void launch_all(const Kv8Cache &c, const Kv8Step &s, const Kv8Attend &a, const Kv8Shape &h, ErrorWord err,
                cudaStream_t stream) {
    constexpr int TERMS = BF16 ? 1 : 2;
    static DeviceOnce once;
    once.run([] {
        cudaFuncSetAttribute(kv8_prompt_kernel<D, BF16, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kPromptSmem<D, TERMS>);
    });
    if (h.prompt_tiles > 0) {
        {
            KernelTimer timer("kv8_prompt", stream);
            launch_pdl(kv8_prompt_kernel<D, BF16, E4M3>, h.prompt_tiles * c.heads * h.prompt_splits, kPromptThreads,
                       kPromptSmem<D, TERMS>, stream, c, s, a, h, err);
            count_launch();
        }
        if (h.prompt_splits > 1) {
            launch_pdl(kv8_join_kernel<D, BF16>, h.prompt_tiles * c.heads * h.prompt_rows, kJoinThreads, 0, stream, c, s, a,
                       h, 1u, err);
            count_launch();
        }
    }
    if constexpr (BF16)
        launch_rows<D, kPlain, E4M3>(c, s, a, h, err, stream);
    else
        h.row_tile == 8 ? launch_rows<D, kStacked, E4M3>(c, s, a, h, err, stream)
                        : launch_rows<D, kTwoTerm, E4M3>(c, s, a, h, err, stream);
    if (h.row_splits > 1) {
        launch_pdl(kv8_join_kernel<D, BF16>, s.requests * h.row_tiles * c.heads * h.join_rows * h.join_chunks, kJoinThreads,
                   0, stream, c, s, a, h, 0u, err);
        count_launch();
    }
}

template <int D>
void launch_typed(const Kv8Cache &c, const Kv8Step &s, const Kv8Attend &a, const Kv8Shape &h, ErrorWord err,
                  cudaStream_t stream) {
    if (a.bf16)
        c.e4m3 ? launch_all<D, true, true>(c, s, a, h, err, stream) : launch_all<D, true, false>(c, s, a, h, err, stream);
    else
        c.e4m3 ? launch_all<D, false, true>(c, s, a, h, err, stream) : launch_all<D, false, false>(c, s, a, h, err, stream);
}

uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

}  // namespace

Kv8Shape kv8_attend_shape(const Kv8Cache &c, const Kv8Step &s, uint32_t query_heads, bool bf16,
                          uint64_t max_kv_length) {
    Kv8Shape h{};
    const uint64_t G = query_heads / c.heads;
    const uint64_t room = (uint64_t)s.columns * c.page_tokens;
    const uint64_t deepest = max_kv_length == 0 ? room : std::min<uint64_t>(max_kv_length, room);
    const uint64_t groups = std::max<uint64_t>(1, ceil_div(deepest, kG));
    // the longest request, if every request brings a token
    const uint64_t longest = (s.tokens > s.requests ? s.tokens - s.requests : 0) + 1, rows = longest * G;
    const bool prompts = rows > kShortRows;
    h.row_tiles = (uint32_t)ceil_div(std::min<uint64_t>(rows, kShortRows), 16);
    h.row_limit = prompts ? kShortRows : UINT32_MAX;
    h.row_tile = !bf16 && rows <= 8 ? 8 : 16;
    // about two waves of two CTAs per SM if every request were the deepest
    const uint64_t items = (uint64_t)s.requests * h.row_tiles * c.heads;
    uint64_t each = ceil_div(items * groups, 4 * kSms);
    each = std::min<uint64_t>(kMaxRowGroups, std::max<uint64_t>(kMinRowGroups, each));
    h.row_groups = (uint32_t)each;
    h.row_splits = (uint32_t)std::min<uint64_t>(ceil_div(groups, each), 4096);
    h.join_rows = (uint32_t)std::min<uint64_t>(rows, 16);
    h.join_chunks = items * h.join_rows < kSms ? c.dim / 64 : 1u;
    h.row_floats = h.row_splits > 1 ? items * h.row_splits * 16 * (c.dim + 2) : 0;
    h.prompt_rows = c.dim == 256 ? kPromptRows<256> : c.dim == 128 ? kPromptRows<128> : kPromptRows<64>;
    if (prompts) {
        h.prompt_tiles = (uint32_t)((uint64_t)s.tokens * G / h.prompt_rows + s.requests);
        const uint64_t work = ceil_div((uint64_t)s.tokens * G, h.prompt_rows) * c.heads;
        const uint64_t cut = std::max<uint64_t>(1, std::min<uint64_t>(ceil_div(2 * kSms, work), 32));
        h.prompt_groups = (uint32_t)(ceil_div(std::max<uint64_t>(kMinPromptGroups, ceil_div(groups, cut)), kPromptGroups) * kPromptGroups);
        h.prompt_splits = work >= kSms ? 1u : (uint32_t)ceil_div(groups, h.prompt_groups);
        h.prompt_floats = h.prompt_splits > 1
                              ? (uint64_t)h.prompt_tiles * c.heads * h.prompt_splits * h.prompt_rows * (c.dim + 2) : 0;
    }
    return h;
}

void launch_kv8_attend(const Kv8Cache &c, const Kv8Step &s, const Kv8Attend &a, const Kv8Shape &shape, ErrorWord err,
                       cudaStream_t stream) {
    if (c.dim == 256)
        launch_typed<256>(c, s, a, shape, err, stream);
    else if (c.dim == 128)
        launch_typed<128>(c, s, a, shape, err, stream);
    else
        launch_typed<64>(c, s, a, shape, err, stream);
}

}  // namespace kqb
