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
// significant bits, exponents -9..8), so the products S = Q K^T and O = P V
// run on the tensor cores with fp16 operands and F32 accumulators.
// A row of Q is scaled by an exact power of two so that its largest element
// lies in [2^13, 2^14): bfloat16 queries are then exact in fp16 (elements
// 2^-27 below the row's largest lose bits, below F32's own rounding of the
// sum), F32 queries are split into two fp16 parts (22 bits).  P sV is scaled
// into fp16's range the same way (below) and split in two for F32 outputs;
// for bfloat16 outputs one part is kept: 11 bits, 2^-11 relative per weight
// against the output's own 2^-8.  The page scales multiply the accumulators
// (sK) and the weights (sV), never the codes.
//
// Softmax in base 2, one pass: a row's reference point m is raised only when
// a logit exceeds it by more than 8, so weights stay below 2^8 and the
// accumulators are rarely rescaled; m, the sums l and O are F32.  The weights
// entering the second product are p * sV against a reference point of their
// own (kernels_kv8.cuh): at most 2^14, the row's largest 2^5 or more, so what
// fp16 cannot hold of a weight is below 2^-30 of the row's largest.
//
// Layout.  A page keeps its codes in the order the fragments need (see
// Kv8Cache), so a warp reads both operands with conflict-free 16-byte shared
// loads and no transposes, and a group of 16 tokens is one contiguous bulk
// copy of 32 * d bytes.
//
// Two kernels:
//   rows     8 or 16 query rows per CTA, for single tokens and short chunks.
//            The rows are the N side of the products (S^T = K Q^T,
//            O^T = V^T P^T), so that 8 rows waste nothing of an
//            m16n8k16 and O takes D / 4 registers a thread.  Four warps take
//            the groups of the CTA's share in turn, each with its own ring of
//            bulk copies and its own softmax state, and merge at the end.
//            The launch is cut into equal shares of all (tile, head, group)
//            units, whatever the requests' lengths; a tile that spans shares
//            leaves (m, l, O) partials which a second kernel joins in order.
//            HBM bound: every (request, head) reads its codes once.
//   prompt   tcgen05 tiles of 128 rows (kernels_kv8_prompt.cu).
// Partials are joined in a fixed order: results do not depend on timing.
#include "kernels_kv8.cuh"

#include <algorithm>

namespace kqb {

namespace {

// Writes ROWS rows from row0 of request `rq` as fragments into q and, per row,
// 1 / its power of two (times the softmax scale in base 2) into factor and its
// last visible token into limit.  Eight threads per row, every thread of the
// CTA takes part; rows behind the request's last are zero with limit -1.
// Returns whether a query value was not finite.
// The rows are the products' N side: [8-row tile][TERMS][D / 16][32 lanes][2].
template <int D, int TERMS, int THREADS, int ROWS>
__device__ __forceinline__ bool load_queries(const Kv8Attend &a, const Request &rq, uint32_t G, uint32_t head,
                                             uint32_t row0, void *q, float *factor, int32_t *limit, uint32_t tid) {
    bool bad = false;
    uint32_t *q32 = static_cast<uint32_t *>(q);
    const uint32_t part = tid & 7;
    for (uint32_t r = tid >> 3; r < ROWS; r += THREADS / 8) {
        const uint32_t row = row0 + r, token = row / G;
        const bool live = token < rq.n;
        float4 x[D / 32];
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (live)
                x[k] = load4<TERMS == 1>(a.q, (uint64_t)(rq.first + token) * a.q_stride + (uint64_t)(head * G + row % G) * D +
                                                  (part + 8 * k) * 4);
        }
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            bad |= !(fabsf(x[k].x) < INFINITY) || !(fabsf(x[k].y) < INFINITY) || !(fabsf(x[k].z) < INFINITY) ||
                   !(fabsf(x[k].w) < INFINITY);
            top = fmaxf(fmaxf(top, fmaxf(fabsf(x[k].x), fabsf(x[k].y))), fmaxf(fabsf(x[k].z), fabsf(x[k].w)));
        }
        // the eight threads of a row are in one warp; rows run out warp by warp
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        // the row's largest element into [2^13, 2^14); 2^-100 is the smallest that is still scaled
        const int e = max((int)(__float_as_uint(top) >> 23), 27) - 127 - 13;
        const float up = __uint_as_float((uint32_t)(127 - e) << 23), down = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            const uint32_t f = (part + 8 * k) * 4, step = f / 64 * 4 + f % 16 / 4, lane = (r & 7) * 4 + f % 64 / 16;
            const float a0 = x[k].x * up, a1 = x[k].y * up, a2 = x[k].z * up, a3 = x[k].w * up;
            const uint32_t h0 = pack_half(a0, a1), h1 = pack_half(a2, a3);
            const uint32_t at = (((r >> 3) * TERMS * (D / 16) + step) * 32 + lane) * 2;
            q32[at] = h0;
            q32[at + 1] = h1;
            if constexpr (TERMS == 2) {
                q32[at + D / 16 * 64] = pack_rest(a0, a1, h0);
                q32[at + D / 16 * 64 + 1] = pack_rest(a2, a3, h1);
            }
        }
        if (part == 0) {
            factor[r] = a.scale_log2 * down;
            limit[r] = live ? (int32_t)(rq.length - rq.n + token) : -1;
        }
    }
    return bad;
}

// ------------------------------------------------------------------- rows

constexpr int kRowWarps = 4, kRowThreads = kRowWarps * 32;
constexpr uint32_t kMinShare = 2 * kRowWarps;   // units: two groups to a warp
// CTAs per SM and ring slots per warp: registers hold NT * D / 4 accumulators
// a thread, shared memory the rings (and, at the end, the warps' merge).
template <int D, int NT> constexpr int kRowCtas = NT * D == 512 ? 2 : D == 256 || NT * D == 256 ? 3 : 4;
template <int D, int NT> constexpr int kRowStages = NT * D == 512 ? 3 : D == 256 ? 2 : NT * D == 256 ? 4 : D == 128 ? 3 : 5;
template <int D, int NT, int TERMS>
constexpr uint32_t kRowSmem = kRowWarps * kRowStages<D, NT> * 32 * D + NT * TERMS * 16 * D;

// A warp's softmax state and accumulators of NT tiles of 8 rows.  Thread (g, t)
// = (lane / 4, lane % 4) holds rows 2t and 2t + 1 of each tile.
template <int D, int NT>
struct Columns {
    float o[NT][D / 16][4];
    float m[NT][2], z[NT][2], l[NT][2];   // reference points m, m + z; sums

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int a = 0; a < NT; ++a) {
#pragma unroll
            for (int r = 0; r < 2; ++r) m[a][r] = z[a][r] = -INFINITY, l[a][r] = 0.0f;
#pragma unroll
            for (int n = 0; n < D / 16; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[a][n][k] = 0.0f;
        }
    }
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// One step over a group of 16 tokens with the rows on the N side.  A key
// fragment's rows are tokens g and g + 8; a value fragment's rows are features
// 4 g + i and 4 g + i + 1 of 32.  The weights come out of the first product
// with tokens as rows and are turned by movmatrix.  The first product runs in
// four chains of MMAs (one chain per group was what this kernel waited for).
template <int D, int NT, int TERMS, bool E4M3, bool MASK>
__device__ __forceinline__ void column_step(Columns<D, NT> &st, const uint2 *q, const uint8_t *kv, float ks, float vs,
                                            const float (&factor)[NT][2], const int32_t (&limit)[NT][2], int32_t token,
                                            uint32_t lane) {
    constexpr int CH = 4 / NT;
    float c[CH][NT][4];
#pragma unroll
    for (int x = 0; x < CH; ++x)
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int k = 0; k < 4; ++k) c[x][a][k] = 0.0f;
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
        const uint4 w0 = *reinterpret_cast<const uint4 *>(kv + j * 1024 + lane * 16);
        const uint4 w1 = *reinterpret_cast<const uint4 *>(kv + j * 1024 + 512 + lane * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint4 x;
            widen<E4M3>(i == 0 ? w0.x : i == 1 ? w0.y : i == 2 ? w0.z : w0.w, x.x, x.z);
            widen<E4M3>(i == 0 ? w1.x : i == 1 ? w1.y : i == 2 ? w1.z : w1.w, x.y, x.w);
#pragma unroll
            for (int a = 0; a < NT; ++a)
#pragma unroll
                for (int term = 0; term < TERMS; ++term) {
                    const uint2 f = q[((a * TERMS + term) * (D / 16) + j * 4 + i) * 32 + lane];
                    mma(c[(i * TERMS + term) % CH][a], x, f.x, f.y);
                }
        }
    }
    float s[NT][4], top[NT][2];
    const float size = size_of(vs);
    bool lift = false;
#pragma unroll
    for (int a = 0; a < NT; ++a) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float v = c[0][a][k];
#pragma unroll
            for (int x = 1; x < CH; ++x) v += c[x][a][k];
            v *= factor[a][k & 1] * ks;
            if (MASK && token + (k >> 1) * 8 + (int32_t)(lane >> 2) > limit[a][k & 1]) v = -INFINITY;
            s[a][k] = v;
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float x = fmaxf(s[a][r], s[a][2 + r]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
            top[a][r] = x;
            lift |= x > st.m[a][r] + kRaise || x - st.m[a][r] + size > st.z[a][r] + kRaise;
        }
    }
    if (__any_sync(~0u, lift)) {   // -inf + 8 is -inf: the first finite logit of a row lifts it
#pragma unroll
        for (int a = 0; a < NT; ++a) {
            float by[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float m = fmaxf(st.m[a][r], ceilf(top[a][r]));
                by[r] = 1.0f;
                if (m == -INFINITY) continue;
                const float less = st.m[a][r] - m, old = st.z[a][r] + less, z = fmaxf(old, ceilf(top[a][r] - m + size));
                st.l[a][r] *= exp2_approx(less);
                by[r] = exp2_approx(old - z);
                st.m[a][r] = m;
                st.z[a][r] = z;
            }
#pragma unroll
            for (int n = 0; n < D / 16; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) st.o[a][n][k] *= by[k & 1];
        }
    }
    uint2 p[NT][TERMS];
#pragma unroll
    for (int a = 0; a < NT; ++a) {
        float e[4];
        const float w[2] = {fminf(weight_of(st.m[a][0], st.z[a][0]) * vs, kMost), fminf(weight_of(st.m[a][1], st.z[a][1]) * vs, kMost)};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            e[k] = exp2_approx(s[a][k] - (st.m[a][k & 1] == -INFINITY ? 0.0f : st.m[a][k & 1]));
            st.l[a][k & 1] += e[k];
            e[k] *= w[k & 1];
        }
        const uint32_t h0 = pack_half(e[0], e[1]), h1 = pack_half(e[2], e[3]);
        p[a][0] = make_uint2(transpose8x8(h0), transpose8x8(h1));
        if constexpr (TERMS == 2)
            p[a][1] = make_uint2(transpose8x8(pack_rest(e[0], e[1], h0)), transpose8x8(pack_rest(e[2], e[3], h1)));
    }
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
        const uint4 v = *reinterpret_cast<const uint4 *>(kv + 16 * D + j * 512 + lane * 16);
        uint4 x[2];
        widen<E4M3>(v.x, x[0].x, x[0].z);
        widen<E4M3>(v.y, x[0].y, x[0].w);
        widen<E4M3>(v.z, x[1].x, x[1].z);
        widen<E4M3>(v.w, x[1].y, x[1].w);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int a = 0; a < NT; ++a)
#pragma unroll
                for (int term = TERMS - 1; term >= 0; --term) mma(st.o[a][j * 2 + i], x[i], p[a][term].x, p[a][term].y);
    }
}

// The row kernel's share of the work.  A unit is one group of one (request,
// tile, head); every tile of a request counts as many as its last one sees.
// The launch's shares are as many as the sizes the host knows can use; of
// these the first `total / kMinShare` work, so that none is empty or tiny.
// The first unit of share k of n over `total` units:
__device__ __forceinline__ uint64_t share_begin(uint64_t total, uint32_t k, uint32_t n) { return total * k / n; }

__device__ __forceinline__ uint32_t row_items(const Request &rq, uint32_t G, uint32_t tile_rows, uint32_t heads,
                                              uint64_t row_limit) {
    const uint64_t rows = (uint64_t)rq.n * G;
    return rows > row_limit ? 0u : (uint32_t)((rows + tile_rows - 1) / tile_rows) * heads;
}

// At least one, so that a request without cached tokens still gets its zeros.
__device__ __forceinline__ uint32_t item_units(const Request &rq) { return max(1u, (rq.length + kG - 1) / kG); }

// What share k leaves for the join: the tile that it begins and does not end.
struct Cut {
    uint32_t request, tile, head, last;   // last: the share that ends it (0: nothing was cut)
};

// A share's partials: [share][ended, begun] of [rows][D] floats, then (m, l)
// per row, then the cuts.
struct ShareSpace {
    float *o;
    float2 *ml;
    Cut *cuts;
    __device__ __forceinline__ ShareSpace(float *base, uint32_t shares, uint32_t rows, uint32_t dim) {
        o = base;
        ml = reinterpret_cast<float2 *>(base + 2ull * shares * rows * dim);
        cuts = reinterpret_cast<Cut *>(ml + 2ull * shares * rows);
    }
};

}  // namespace

// grid: equal shares of all units.  Each warp streams every fourth group of a
// tile through its own ring; page ids and scales of its next 64 groups sit in
// its lanes.
// Measured: 64 F32 sequences, contexts U[1k, 32k], 16 heads of 256 over int8
// pages: 1086 MB in 191 to 203 us, by machine, with the join (5.7 to 5.3 TB/s of the
// measured 6.5; under ncu the kernel alone 173 to 180 us); 96 bf16 sequences up to 8k, 32 heads of 128 over
// e4m3 pages: 892 MB in 160 to 166 us.  (16 rows on the M side, one split per 2048
// tokens and a join kernel per row: 244 and 242 us.)
template <int D, int NT, int TERMS, bool E4M3>
__global__ void __launch_bounds__(kRowThreads, (kRowCtas<D, NT>))
kv8_rows_kernel(Kv8Cache c, Kv8Step s, Kv8Attend a, Kv8Shape shape, ErrorWord err) {
    constexpr int ST = kRowStages<D, NT>;
    constexpr bool BF16 = TERMS == 1;
    constexpr uint32_t kStage = 32 * D, kRows = 8 * NT;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[kRowWarps][ST];
    __shared__ float factor_s[kRows], merge_m[kRowWarps][kRows], merge_l[kRowWarps][kRows];
    __shared__ int32_t limit_s[kRows];
    __shared__ uint64_t warp_units[kRowWarps], begin_unit;
    __shared__ uint32_t begin_request;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint8_t *ring = smem + warp * ST * kStage;
    uint2 *q = reinterpret_cast<uint2 *>(smem + kRowWarps * ST * kStage);
    const uint32_t G = a.query_heads / c.heads, share = blockIdx.x, shares = gridDim.x;
    const ShareSpace space(a.workspace, shares, kRows, D);

    if (tid < kRowWarps * ST) bar_init(&full[0][0] + tid, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    pdl_wait();
    // before any way out: the join reads every share's cut, and the error that
    // ends this kernel may be cleared before the join looks (a graph's replay on
    // one stream, a synchronize of another)
    if (shares > 1 && tid == 0) space.cuts[share].last = 0;
    if (__syncthreads_or(tid == 0 && err_raised(err))) return;

    // units of all requests: consecutive requests per thread, then the request
    // in which this share begins
    Request rq;
    const uint32_t per = (s.requests + kRowThreads - 1) / kRowThreads;
    const uint32_t b0 = min(tid * per, s.requests), b1 = min(b0 + per, s.requests);
    uint64_t units = 0;
    bool good = true;
    for (uint32_t b = b0; b < b1; ++b)
        if (load_request(c, s, b, rq, err))
            units += (uint64_t)row_items(rq, G, kRows, c.heads, shape.row_limit) * item_units(rq);
        else
            good = false;
    uint64_t upto = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(~0u, upto, o);
        if (lane >= (uint32_t)o) upto += x;
    }
    if (lane == 31) warp_units[warp] = upto;
    if (__syncthreads_or(!good)) return;
    uint64_t total = 0;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
        if (w < (int)warp) upto += warp_units[w];
        total += warp_units[w];
    }
    const uint32_t working = (uint32_t)min((uint64_t)shares, max(total / kMinShare, (uint64_t)1));
    if (share >= working || total == 0) return;
    uint64_t at = share_begin(total, share, working);
    const uint64_t end = share_begin(total, share + 1, working);
    if (at >= upto - units && at < upto) {
        uint64_t left = at - (upto - units);
        for (uint32_t b = b0; b < b1; ++b) {
            load_request(c, s, b, rq, err);
            const uint64_t n = (uint64_t)row_items(rq, G, kRows, c.heads, shape.row_limit) * item_units(rq);
            if (left < n) {
                begin_request = b;
                begin_unit = left;
                break;
            }
            left -= n;
        }
    }
    __syncthreads();
    uint32_t b = begin_request;
    uint64_t inside = begin_unit;   // unit of request b
    load_request(c, s, b, rq, err);

    uint32_t used = 0;   // ring slots used so far (waits go by it)
    while (true) {
        const uint32_t depth = item_units(rq), item = (uint32_t)(inside / depth), u0 = (uint32_t)(inside % depth);
        const uint32_t tile = item / c.heads, head = item % c.heads;
        const uint32_t u1 = (uint32_t)min((uint64_t)depth, u0 + (end - at));
        const uint32_t rows = rq.n * G, row0 = tile * kRows, row_end = min(row0 + kRows, rows);
        const uint32_t groups = visible_groups(rq, G, row_end), g0 = min(u0, groups), g1 = min(u1, groups);
        const int32_t *table = s.table + (uint64_t)b * s.table_stride;
        const uint32_t per_page = c.page_tokens / kG;
        const uint64_t page_bytes = 2ull * c.page_tokens * D;
        // this warp's groups: g0 + warp + 4 i
        const uint32_t mine = g1 > g0 + warp ? (g1 - g0 - warp + kRowWarps - 1) / kRowWarps : 0;
        uint32_t page[2] = {0, 0};   // page ids and scales of 32 groups, and of the next 32
        float2 scales[2] = {};
        auto fetch = [&](uint32_t from, int k) {
            const uint32_t i = from + lane;
            if (i < mine) {
                const int32_t id = table[(g0 + warp + i * kRowWarps) / per_page];
                const bool ok = id >= 0 && (uint32_t)id < c.pages;
                if (!ok) raise(err, kErrStep);
                page[k] = ok ? (uint32_t)id : 0u;   // any page: the call fails
                scales[k] = *reinterpret_cast<const float2 *>(c.scales + ((uint64_t)page[k] * c.heads + head) * 2);
            }
        };
        auto issue = [&](uint32_t i, uint32_t from) {   // group i of this warp into its slot; lanes hold from .. from + 63
            const uint32_t id = __shfl_sync(~0u, i - from < 32 ? page[0] : page[1], i & 31);
            if (lane == 0) {
                const uint32_t slot = (used + i) % ST;
                bar_expect(&full[warp][slot], kStage);
                bulk_copy(ring + slot * kStage,
                          c.codes + ((uint64_t)id * c.heads + head) * page_bytes +
                              (uint64_t)((g0 + warp + i * kRowWarps) % per_page) * kStage,
                          kStage, &full[warp][slot]);
            }
        };
        fetch(0, 0);
        uint32_t issued = 0;
        for (; issued < min(mine, (uint32_t)ST); ++issued) issue(issued, 0);
        fetch(32, 1);

        if (load_queries<D, TERMS, kRowThreads, kRows>(a, rq, G, head, row0, q, factor_s, limit_s, tid))
            raise(err, kErrNonFinite);
        __syncthreads();
        Columns<D, NT> st;
        st.clear();
        float factor[NT][2];
        int32_t limit[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                factor[n][r] = factor_s[n * 8 + (lane & 3) * 2 + r];
                limit[n][r] = limit_s[n * 8 + (lane & 3) * 2 + r];
            }
        // every row of the tile sees the tokens before this one
        const uint32_t clear_to = row_end == row0 + kRows && rq.length + 1 > rq.n ? rq.length - rq.n + row0 / G + 1 : 0u;
        bool ok = true;
        uint32_t i = 0;
        for (; i < mine; ++i) {
            if (i > 0 && (i & 31) == 0) {
                page[0] = page[1];
                scales[0] = scales[1];
                fetch(i + 32, 1);
            }
            const uint32_t slot = (used + i) % ST;
            ok = bar_wait_warp(&full[warp][slot], (used + i) / ST & 1u);
            if (!ok) break;
            const float ks = __shfl_sync(~0u, scales[0].x, i & 31), vs = __shfl_sync(~0u, scales[0].y, i & 31);
            const uint32_t token = (g0 + warp + i * kRowWarps) * kG;
            const uint8_t *kv = ring + slot * kStage;
            if (token + kG > clear_to)
                column_step<D, NT, TERMS, E4M3, true>(st, q, kv, ks, vs, factor, limit, (int32_t)token, lane);
            else
                column_step<D, NT, TERMS, E4M3, false>(st, q, kv, ks, vs, factor, limit, (int32_t)token, lane);
            __syncwarp();
            if (issued < mine) issue(issued++, i & ~31u);
        }
        if (!ok) {
            // a wait gave up: let the other copies land before the CTA exits
            if (lane == 0) raise(err, kErrTimeout);
            for (uint32_t k = i; k < issued; ++k) bar_wait_warp(&full[warp][(used + k) % ST], (used + k) / ST & 1u);
        }
        used += mine;

        // join the warps: (m, l) and O of each in its own ring
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float l = st.l[n][r];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(~0u, l, o);
                if (lane < 4) {
                    merge_m[warp][n * 8 + lane * 2 + r] = st.m[n][r];
                    merge_l[warp][n * 8 + lane * 2 + r] = l;
                }
            }
        constexpr uint32_t kPitch = D + 4;   // rows 4 banks apart: conflict-free 16-byte stores
        float *mo = reinterpret_cast<float *>(ring);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float back = back_of(st.m[n][r], st.z[n][r]);
#pragma unroll
                for (int j = 0; j < D / 32; ++j)
                    *reinterpret_cast<float4 *>(mo + (n * 8 + (lane & 3) * 2 + r) * kPitch + j * 32 + (lane >> 2) * 4) =
                        make_float4(st.o[n][2 * j][r] * back, st.o[n][2 * j][2 + r] * back, st.o[n][2 * j + 1][r] * back,
                                    st.o[n][2 * j + 1][2 + r] * back);
            }
        __syncthreads();
        const bool begun = u0 == 0, ended = u1 == depth;
        const uint64_t place = 2ull * share + (begun ? 1 : 0);   // of a partial
        for (uint32_t v = tid; v < (row_end - row0) * (D / 4); v += kRowThreads) {
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
            if (begun && ended) {
                finish4<BF16>(a, rq, G, head, row0 + r, f, D, m, l, o, err);
            } else {
                *reinterpret_cast<float4 *>(space.o + (place * kRows + r) * D + f) = o;
                if (f == 0) space.ml[place * kRows + r] = make_float2(m, l);
            }
        }
        if (begun && !ended && tid == 0)
            space.cuts[share] = {b, tile, head, (uint32_t)(((at + (depth - u0)) * working - 1) / total)};
        // the ring's next writes come through the asynchronous proxy
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (__syncthreads_or(!ok)) return;
        at += u1 - u0;
        if (at >= end) return;
        inside += u1 - u0;
        // the next request that has units (there is one: at < end)
        while (inside >= (uint64_t)row_items(rq, G, kRows, c.heads, shape.row_limit) * depth || rq.n == 0) {
            inside = 0;
            if (++b >= s.requests) return;
            load_request(c, s, b, rq, err);
            if (row_items(rq, G, kRows, c.heads, shape.row_limit) > 0) break;
            rq.n = 0;
        }
    }
}

namespace {

constexpr int kShareJoinThreads = 256;

}  // namespace

// Joins the tiles that shares cut, from shares k (which began it) .. last in
// this order.  Narrow: CTA k takes the tile that share k began, a thread per 4
// features.  WIDE, for few tiles of many partials: CTA (i, chunk) takes the
// i-th such tile, of it 64 features of one row, the partials dealt to 16
// groups of 16 threads.
// Bound: latency, the partials come from L2.
template <int D, int NT, bool BF16, bool WIDE>
__global__ void __launch_bounds__(kShareJoinThreads)
kv8_rows_join_kernel(Kv8Cache c, Kv8Step s, Kv8Attend a, Kv8Shape shape, ErrorWord err) {
    constexpr uint32_t kRows = 8 * NT, kCells = kRows * (D / 4);
    constexpr uint32_t kChunks = WIDE ? kRows * (D / 64) : 1, kWays = WIDE ? 16 : 1, kAhead = 8;
    constexpr uint32_t kPer = 3;   // shares per thread of the search (at most 592 shares)
    __shared__ float4 way_o[kWays][WIDE ? 16 : 1];
    __shared__ float way_m[kWays], way_l[kWays];
    __shared__ uint32_t warp_cuts[kShareJoinThreads / 32], found;
    const uint32_t tid = threadIdx.x, chunk = blockIdx.x % kChunks;
    const uint32_t G = a.query_heads / c.heads;
    pdl_wait();
    if (__syncthreads_or(tid == 0 && err_raised(err))) return;
    const ShareSpace space(a.workspace, shape.row_shares, kRows, D);
    const uint32_t way = WIDE ? tid / 16 : 0u;
    auto join = [&](uint32_t share) {   // every thread of the CTA
        const Cut cut = space.cuts[share];
        Request rq;
        if (cut.last <= share || !load_request(c, s, cut.request, rq, err)) return;
        const uint32_t row0 = cut.tile * kRows, row_end = min(row0 + kRows, rq.n * G), n = cut.last - share + 1;
        for (uint32_t v = WIDE ? chunk * 16 + tid % 16 : tid; v < kCells; v += WIDE ? kCells : kShareJoinThreads) {
            const uint32_t r = v / (D / 4), f = v % (D / 4) * 4;
            if (row0 + r >= row_end) break;
            float m = -INFINITY, l = 0.0f;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (uint32_t k = way; k < n; k += kWays * kAhead) {
                float4 y[kAhead];
                float2 x[kAhead];
#pragma unroll
                for (uint32_t i = 0; i < kAhead; ++i) {
                    const uint32_t at = k + i * kWays;
                    // the first share's partial is the one it began, the others' the one they ended or passed through
                    const uint64_t place = 2ull * (share + at) + (at == 0 ? 1 : 0);
                    const bool in = at < n;
                    y[i] = in ? *reinterpret_cast<const float4 *>(space.o + (place * kRows + r) * D + f)
                              : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    x[i] = in ? space.ml[place * kRows + r] : make_float2(-INFINITY, 0.0f);
                }
                float top = m;
#pragma unroll
                for (uint32_t i = 0; i < kAhead; ++i) top = fmaxf(top, x[i].x);
                if (top == -INFINITY) continue;
                const float by = exp2_approx(m - top);
                m = top;
                l *= by, o.x *= by, o.y *= by, o.z *= by, o.w *= by;
#pragma unroll
                for (uint32_t i = 0; i < kAhead; ++i) {
                    const float w = exp2_approx(x[i].x - m);
                    l += x[i].y * w;
                    o.x += y[i].x * w, o.y += y[i].y * w, o.z += y[i].z * w, o.w += y[i].w * w;
                }
            }
            if constexpr (WIDE) {   // all threads are on the same row
                way_o[way][tid % 16] = o;
                if (tid % 16 == 0) way_m[way] = m, way_l[way] = l;
                __syncthreads();
                m = way_m[0];
#pragma unroll
                for (uint32_t w = 1; w < kWays; ++w) m = fmaxf(m, way_m[w]);
                l = 0.0f;
                o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (uint32_t w = 0; w < kWays; ++w) {
                    const float by = way_m[w] == -INFINITY ? 0.0f : exp2_approx(way_m[w] - m);
                    const float4 y = way_o[w][tid % 16];
                    l += way_l[w] * by;
                    o.x += y.x * by, o.y += y.y * by, o.z += y.z * by, o.w += y.w * by;
                }
            }
            if (way == 0) finish4<BF16>(a, rq, G, cut.head, row0 + r, f, D, m, l, o, err);
        }
    };
    if constexpr (!WIDE) {
        join(blockIdx.x);
    } else {
        uint32_t cuts = 0;
#pragma unroll
        for (uint32_t k = tid * kPer; k < tid * kPer + kPer; ++k) cuts += k < shape.row_shares && space.cuts[k].last > k;
        uint32_t before = cuts, total = 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(~0u, before, o);
            if ((tid & 31) >= (uint32_t)o) before += x;
        }
        if ((tid & 31) == 31) warp_cuts[tid >> 5] = before;
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < kShareJoinThreads / 32; ++w) {
            if (w < tid / 32) before += warp_cuts[w];
            total += warp_cuts[w];
        }
        before -= cuts;
        // one tile per CTA, unless requests have more tiles than the launch expected
        for (uint32_t want = blockIdx.x / kChunks; want < total; want += shape.join_tiles) {
            if (want >= before && want < before + cuts) {
                uint32_t left = want - before;
                for (uint32_t k = tid * kPer; k < tid * kPer + kPer; ++k)
                    if (k < shape.row_shares && space.cuts[k].last > k && left-- == 0) found = k;
            }
            __syncthreads();
            join(found);
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------ prompt join

namespace {

constexpr int kJoinThreads = 256;

}  // namespace

// Joins the splits of a prompt tile: one CTA per (tile, head, 16 rows), a
// thread per 4 features of a row, in split order.
template <int D, bool BF16>
__global__ void __launch_bounds__(kJoinThreads)
kv8_prompt_join_kernel(Kv8Cache c, Kv8Step s, Kv8Attend a, Kv8Shape shape, ErrorWord err) {
    constexpr uint32_t kAhead = 8;
    const uint32_t tid = threadIdx.x, G = a.query_heads / c.heads, kRows = shape.prompt_rows;
    const uint32_t block = blockIdx.x % (kRows / 16), u = blockIdx.x / (kRows / 16), head = u % c.heads, t = u / c.heads;
    pdl_wait();
    if (__syncthreads_or(tid == 0 && err_raised(err))) return;
    uint32_t start;
    const uint32_t b = find_request(s, G, kRows, t, tid & 31, start);
    Request rq;
    if (t < start || !load_request(c, s, b, rq, err)) return;
    const uint64_t rows64 = (uint64_t)rq.n * G;
    if (rows64 <= shape.row_limit || (uint64_t)(t - start) * kRows >= rows64) return;
    const uint32_t rows = (uint32_t)rows64, row0 = (t - start) * kRows, row_end = min(row0 + kRows, rows);
    const uint32_t groups = visible_groups(rq, G, row_end);
    const uint32_t each = split_groups(groups, shape.prompt_groups, shape.prompt_splits, kPromptUnit);
    if (groups <= each) return;
    const uint32_t n = (groups + each - 1) / each;
    const Partials part(a.workspace + shape.row_floats, (uint64_t)t * c.heads + head, shape.prompt_splits, kRows, D,
                        (uint64_t)shape.prompt_tiles * c.heads);
    for (uint32_t v = tid; v < 16 * (D / 4); v += kJoinThreads) {
        const uint32_t r = block * 16 + v / (D / 4), f = v % (D / 4) * 4;
        if (row0 + r >= row_end) break;
        const float2 *ml = part.ml + (uint64_t)r * shape.prompt_splits;
        const float *po = part.o + (uint64_t)r * D + f;
        float m = -INFINITY, l = 0.0f;
        for (uint32_t k = 0; k < n; ++k) m = fmaxf(m, ml[k].x);
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (uint32_t k = 0; k < n; k += kAhead) {
            float4 y[kAhead];
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i)
                y[i] = k + i < n ? *reinterpret_cast<const float4 *>(po + (uint64_t)(k + i) * kRows * D)
                                 : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i) {
                const float2 x = k + i < n ? ml[k + i] : make_float2(-INFINITY, 0.0f);
                const float w = x.x == -INFINITY ? 0.0f : exp2_approx(x.x - m);
                l += x.y * w;
                o.x += y[i].x * w, o.y += y[i].y * w, o.z += y[i].z * w, o.w += y[i].w * w;
            }
        }
        finish4<BF16>(a, rq, G, head, row0 + r, f, D, m, l, o, err);
    }
}

// --------------------------------------------------------------- launching

namespace {

constexpr uint32_t kSms = 148;
// Requests of up to this many rows go to the row kernel.  8 requests over 8k
// cached tokens, row / prompt kernel: F32, 2 heads of 256: 64 rows 88 / 100 us,
// 128 rows 143 / 107; bf16, 8 heads of 128: 119 / 170 and 213 / 178.
constexpr uint32_t kShortRows = 64;
// Steps of at most this many units (as the launch sees them: capacities, not
// lengths) go to the row kernel whole: a prompt tile takes 19 us at least, the
// row kernel 8 us and about 1.7 ns a unit.  Two chunks over 256, 1k, 4k and 8k
// cached tokens, row / prompt kernel: F32, 24 tokens, 2 heads of 256 (960, 3264,
// 12480, 24768 units) 27 / 43, 31 / 88, 47 / 90, 70 / 96 us; bf16, 40 tokens, 8
// heads of 128 over 256, 1k, 4k (3200, 10880, 41600) 20 / 35, 29 / 57, 51 / 61.
// With so few tiles the row kernel is ahead past the limit too; with many it is
// not (8 requests of 128 rows, 65920 units: 143 / 107).
constexpr uint64_t kFewUnits = 8192;
// Shares per tile from which a tile is joined by many CTAs.  Many / one, F32, 2
// heads of 256: one request of 4k, 32k, 131k tokens (32, 222, 222 shares a tile)
// 16 / 22, 25 / 61, 45 / 82 us; 8, 16, 32 of 8k (28, 14, 7) 37 / 39, 53 / 49,
// 84 / 72; bf16, 8 heads of 128: 8 of 8k (9) 49 / 45.
constexpr uint32_t kManyPartials = 8;
// A split of a prompt: this many groups (1024 tokens) or more.  One F32 request,
// 2 heads of 256, with 16, 32, 64 and 256: 128 tokens over 2k 57, 61, 90, 145 us;
// over 16k 205, 205, 180, 250; bf16, 8 heads of 128, 32 tokens over 4k 45, 45,
// 53, 123; over 16k 84, 84, 61, 124: short splits win over short contexts, and
// lose to their joins over long ones.
constexpr uint32_t kMinPromptGroups = 64;

template <int D, int NT, bool BF16, bool E4M3>
void launch_rows(const Kv8Cache &c, const Kv8Step &s, const Kv8Attend &a, const Kv8Shape &h, ErrorWord err,
                 cudaStream_t stream) {
    constexpr int TERMS = BF16 ? 1 : 2;
    static DeviceOnce once;
    once.run([] {
        cudaFuncSetAttribute(kv8_rows_kernel<D, NT, TERMS, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kRowSmem<D, NT, TERMS>);
    });
    {
        KernelTimer timer("kv8_rows", stream);
        launch_pdl(kv8_rows_kernel<D, NT, TERMS, E4M3>, h.row_shares, kRowThreads, kRowSmem<D, NT, TERMS>, stream, c, s, a, h,
                   err);
        count_launch();
    }
    if (h.row_shares > 1) {
        if (h.join_tiles > 0)
            launch_pdl(kv8_rows_join_kernel<D, NT, BF16, true>, h.join_tiles * 8 * NT * (D / 64), kShareJoinThreads, 0, stream, c,
                       s, a, h, err);
        else
            launch_pdl(kv8_rows_join_kernel<D, NT, BF16, false>, h.row_shares, kShareJoinThreads, 0, stream, c, s, a, h, err);
        count_launch();
    }
}

template <int D, bool BF16, bool E4M3>
void launch_all(const Kv8Cache &c, const Kv8Step &s, const Kv8Attend &a, const Kv8Shape &h, ErrorWord err,
                cudaStream_t stream) {
    if (h.prompt_tiles > 0) {
        launch_kv8_prompt(c, s, a, h, err, stream);
        if (h.prompt_splits > 1) {
            launch_pdl(kv8_prompt_join_kernel<D, BF16>, h.prompt_tiles * c.heads * (h.prompt_rows / 16), kJoinThreads, 0,
                       stream, c, s, a, h, err);
            count_launch();
        }
    }
    h.row_tile == 8 ? launch_rows<D, 1, BF16, E4M3>(c, s, a, h, err, stream)
                    : launch_rows<D, 2, BF16, E4M3>(c, s, a, h, err, stream);
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
    // lengths are 32-bit: no request has more, however wide the table
    const uint64_t room = std::min<uint64_t>((uint64_t)s.columns * c.page_tokens, INT32_MAX);
    const uint64_t deepest = max_kv_length == 0 ? room : std::min<uint64_t>(max_kv_length, room);
    const uint64_t groups = std::max<uint64_t>(1, ceil_div(deepest, kG));
    // the longest request, if every request brings a token
    const uint64_t longest = (s.tokens > s.requests ? s.tokens - s.requests : 0) + 1, rows = longest * G;
    // 16-row groups that the row kernel would walk if it took everything: strips * groups
    const uint64_t strips = ceil_div((uint64_t)s.tokens * G, 16) * c.heads;
    const bool prompts = rows > kShortRows && strips > kFewUnits / groups;
    h.row_limit = prompts ? kShortRows : UINT32_MAX;
    h.row_tile = rows <= 8 ? 8 : 16;
    // one wave of the row kernel, or shares of at least kMinShare groups
    const uint64_t tiles = ceil_div(prompts ? std::min<uint64_t>(rows, kShortRows) : rows, h.row_tile);
    const uint64_t items = s.requests * tiles * c.heads;
    const uint32_t wide = h.row_tile / 8 * c.dim;
    const uint64_t wave = kSms * (wide == 512 ? 2 : c.dim == 256 || wide == 256 ? 3 : 4);
    h.row_shares = (uint32_t)std::min<uint64_t>(wave, std::max<uint64_t>(1, items * groups / kMinShare));
    h.join_tiles = items * kManyPartials <= h.row_shares ? (uint32_t)items : 0;
    h.row_floats = h.row_shares > 1 ? 2ull * h.row_shares * h.row_tile * (c.dim + 2) + 4ull * h.row_shares : 0;
    h.row_floats = ceil_div(h.row_floats, 4) * 4;   // what follows is read 16 bytes at a time
    h.prompt_rows = kv8_prompt_rows(c.dim, bf16);
    if (prompts) {
        h.prompt_tiles = (uint32_t)((uint64_t)s.tokens * G / h.prompt_rows + s.requests);
        const uint64_t work = ceil_div((uint64_t)s.tokens * G, h.prompt_rows) * c.heads;
        const uint64_t cut = std::max<uint64_t>(1, std::min<uint64_t>(ceil_div(2 * kSms, work), 32));
        h.prompt_groups = (uint32_t)(ceil_div(std::max<uint64_t>(kMinPromptGroups, ceil_div(groups, cut)), kPromptUnit) * kPromptUnit);
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
