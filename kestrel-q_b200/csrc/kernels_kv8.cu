// Paged 8-bit key/value cache: the plan of a ragged step, the append of new
// rows and the read-out of pages.  (The attention: kernels_kv8_attend.cu.)
#include "kernels_kv8.cuh"

#include <algorithm>
#include <type_traits>

#include <cuda_fp8.h>

namespace kqb {

namespace {

// go(integral constant) for the head dimension: the layout's divisions are shifts then
template <class Go>
void by_dimension(uint32_t dim, Go go) {
    if (dim == 256)
        go(std::integral_constant<int, 256>());
    else if (dim == 128)
        go(std::integral_constant<int, 128>());
    else
        go(std::integral_constant<int, 64>());
}

// ------------------------------------------------------------------- plan

constexpr int kPlanThreads = 512;
constexpr int kPlanTokens = 4;   // tokens per thread

}  // namespace

// With c_b cached and n_b new tokens of request b, P tokens to a page:
//   off_b   = n_0 + .. + n_{b-1}                        query offsets
//   taken_b = ceil((c_b + n_b) / P) - ceil(c_b / P)     pages from the free list
//   runs_b  = ceil((c_b + n_b) / P) - floor(c_b / P)    (request, page) pairs written
// and token off_b + i sits at position c_b + i.  Every CTA forms the three
// prefix sums of all requests in shared memory (8 bytes read per request, so
// repeating it costs less than a second launch) and fills its own range of
// tokens: one binary search per token.  A page that the step takes from the
// free list begins with one of its tokens, and that token's thread writes the
// table entry; the others compute the id from the same prefix sum, so no
// thread reads what another writes.
// Bound: latency: 6.1 us under ncu for 64 decode requests, 10 us for 512 ragged
// prompts of 119k tokens, caches cold; back to back a call takes 8 us, the host's
// part of it.
__global__ void __launch_bounds__(kPlanThreads)
kv8_plan_kernel(Kv8Cache c, Kv8Step s, Kv8Plan p, ErrorWord err) {
    extern __shared__ int32_t plan_smem[];
    __shared__ long long warp_sum[3][kPlanThreads / 32];
    const uint32_t B = s.requests, P = c.page_tokens, tid = threadIdx.x;
    int32_t *off = plan_smem, *taken = off + B + 1, *runs = taken + B + 1;
    pdl_wait();
    if (__syncthreads_or(tid == 0 && err_raised(err))) return;

    // consecutive requests per thread; sums in 64 bits until they are checked
    const uint32_t per = (B + kPlanThreads - 1) / kPlanThreads;
    const uint32_t b0 = min(tid * per, B), b1 = min(b0 + per, B);
    const long long room = (long long)s.columns * P;
    long long sum[3] = {0, 0, 0};
    bool bad = false;
    for (uint32_t b = b0; b < b1; ++b) {
        const int32_t ctx = p.context[b], n = p.fresh[b];
        bad |= ctx < 0 || n < 0 || (long long)ctx + n > room || (long long)ctx + n > INT32_MAX;
        if (bad) break;
        const uint32_t end = ((uint32_t)ctx + n + P - 1) / P;
        off[b] = (int32_t)min(sum[0], (long long)INT32_MAX);
        taken[b] = (int32_t)min(sum[1], (long long)INT32_MAX);
        runs[b] = (int32_t)min(sum[2], (long long)INT32_MAX);
        sum[0] += n;
        sum[1] += end - ((uint32_t)ctx + P - 1) / P;
        sum[2] += n > 0 ? end - (uint32_t)ctx / P : 0u;
    }
    const uint32_t lane = tid & 31, warp = tid >> 5;
    long long inc[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        long long v = sum[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(~0u, v, o);
            if (lane >= (uint32_t)o) v += u;
        }
        inc[k] = v;
        if (lane == 31) warp_sum[k][warp] = v;
    }
    bad = __syncthreads_or(bad);
    long long total[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        long long base = 0, all = 0;
#pragma unroll
        for (int w = 0; w < kPlanThreads / 32; ++w) {
            if (w < (int)warp) base += warp_sum[k][w];
            all += warp_sum[k][w];
        }
        inc[k] += base - sum[k];
        total[k] = all;
    }
    const long long head = p.free_head[0];
    bad |= total[0] > s.tokens || total[2] > s.runs || head < 0 || head + total[1] > p.free_count;
    if (bad) {   // the same for every thread of every CTA: nothing is written
        if (tid == 0) raise(err, kErrStep);
        return;
    }
    for (uint32_t b = b0; b < b1; ++b) {
        off[b] += (int32_t)inc[0];
        taken[b] += (int32_t)inc[1];
        runs[b] += (int32_t)inc[2];
        if (blockIdx.x == 0) {
            s.query_offsets[b] = off[b];
            s.run_offsets[b] = runs[b];
            s.kv_lengths[b] = p.context[b] + p.fresh[b];
        }
    }
    if (tid == 0) {
        off[B] = (int32_t)total[0];
        if (blockIdx.x == 0) {
            s.query_offsets[B] = (int32_t)total[0];
            s.run_offsets[B] = (int32_t)total[2];
            p.free_head_out[0] = (int32_t)(head + total[1]);
        }
    }
    __syncthreads();

#pragma unroll
    for (int k = 0; k < kPlanTokens; ++k) {
        const uint32_t t = (blockIdx.x * kPlanTokens + k) * kPlanThreads + tid;
        // page runs behind the last one are marked empty
        if (t < s.runs && t >= (uint32_t)total[2]) s.page_runs[t] = -1;
        if (t >= s.tokens) continue;
        if (t >= (uint32_t)total[0]) {
            s.slots[t] = -1;
            s.positions[t] = -1;
            continue;
        }
        // the last request that begins at or before t (empty ones begin where
        // the next one does)
        uint32_t lo = 0, hi = B;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if ((uint32_t)off[mid] <= t) lo = mid; else hi = mid;
        }
        const uint32_t ctx = (uint32_t)p.context[lo], pos = ctx + (t - (uint32_t)off[lo]);
        const uint32_t column = pos / P, first = (ctx + P - 1) / P;
        int32_t *entry = s.table + (uint64_t)lo * s.table_stride + column;
        const bool fresh = column >= first;
        const int32_t page = fresh ? p.free_pages[head + taken[lo] + (column - first)] : *entry;
        const bool ok = page >= 0 && (uint32_t)page < c.pages;
        if (!ok) raise(err, kErrStep);
        if (ok && fresh && pos % P == 0) *entry = page;
        s.slots[t] = ok ? (int64_t)page * P + pos % P : -1;
        s.positions[t] = (int32_t)pos;
        if (t == (uint32_t)off[lo] || pos % P == 0) s.page_runs[runs[lo] + (column - ctx / P)] = (int32_t)t;
    }
}

void launch_kv8_plan(const Kv8Cache &c, const Kv8Step &s, const Kv8Plan &p, ErrorWord err, cudaStream_t stream) {
    static DeviceOnce once;
    once.run([] {
        cudaFuncSetAttribute(kv8_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             3 * (kKv8MaxRequests + 1) * (int)sizeof(int32_t));
    });
    KernelTimer timer("kv8_plan", stream);
    const uint32_t each = kPlanThreads * kPlanTokens;
    const uint32_t grid = std::max(1u, (std::max(s.tokens, s.runs) + each - 1) / each);
    launch_pdl(kv8_plan_kernel, grid, kPlanThreads, 3 * (s.requests + 1) * sizeof(int32_t), stream, c, s, p, err);
    count_launch();
}

// ----------------------------------------------------------------- append

namespace {

constexpr int kAppendThreads = 256;
constexpr uint32_t kAhead = 4;

// The stored byte of an F32 quotient: nearest, ties to even, clamped to the
// format's range (a scale that is itself subnormal can be rounded down).
template <bool E4M3>
__device__ __forceinline__ uint32_t encode(float q) {
    if constexpr (E4M3) {
        return (uint32_t)__nv_cvt_float_to_fp8(fminf(fmaxf(q, -448.0f), 448.0f), __NV_SATFINITE, __NV_E4M3);
    } else {
        return (uint32_t)(__float2int_rn(fminf(fmaxf(q, -127.0f), 127.0f)) + 128);
    }
}

// Four new values -> four stored bytes, from two products each: with inv the
// rounded 1 / s, low = inv (1 - 2^-22) and high = inv (1 + 2^-22) hold the
// correctly rounded quotient x / s between them, and rounding to the format
// keeps that order.  So where both give one code it is the quotient's; `near`
// is set where they differ (the caller divides then).
// int8: adding 1.5 * 2^23 + 128 rounds the product to an integer, ties to even,
// and leaves its low byte with 128 added.  (Dividing every value: 80 us for 48
// ragged F32 prompts, 50k tokens; this: 60.)
template <bool E4M3>
__device__ __forceinline__ uint32_t encode4(float4 x, float low, float high, bool &near) {
    const uint64_t xy = pack2(x.x, x.y), zw = pack2(x.z, x.w);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint64_t by = i == 0 ? pack2(low, low) : pack2(high, high);
        float a, b, c, d;
        if constexpr (E4M3) {
            unpack2(mul2(xy, by), a, b), unpack2(mul2(zw, by), c, d);
            w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) |
                   (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16;
        } else {
            const uint64_t to = pack2(12583040.0f, 12583040.0f);
            unpack2(fma2(xy, by, to), a, b), unpack2(fma2(zw, by, to), c, d);
            w[i] = __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040),
                               __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
        }
    }
    near |= w[0] != w[1];
    return w[0];
}

template <bool E4M3>
__device__ __forceinline__ float decode(uint32_t byte) {
    if constexpr (E4M3) {
        const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
        return __half2float(__half(h));
    } else {
        return (float)((int)byte - 128);
    }
}

template <bool E4M3> constexpr float kLargest = E4M3 ? 448.0f : 127.0f;
template <bool E4M3> constexpr uint32_t kZeroByte = E4M3 ? 0u : 128u;

}  // namespace

// One CTA per (page run, head, key or value): the run's rows are consecutive
// tokens whose slots lie in one page.  With s' the page's scale (0 for a run
// that begins its page) and m the run's largest magnitude,
//   s = max(s', m / M),   M = 127 (int8) or 448 (e4m3)
// new rows are stored as round(x / s); where s > s', rows before the run are
// stored again as round(code * (s' / s)).  Each quotient is one correctly
// rounded division, so the codes are a function of the rows alone.
// The rows are read twice, for m and for the codes: the second read hits L2
// (a run is at most 128 rows of 1 KB), so HBM sees each row once.
// Each thread makes 16 bytes of the page layout: one key row's 16 features,
// or 4 value features of 4 tokens; a warp's 32 units are 512 contiguous bytes.
// Bound: HBM and the instructions of the rounding for prompts, latency for
// single tokens (one group of 16 tokens is touched unless the scale grows).
// Measured under ncu, caches cold: 48 ragged F32 prompts, 50k tokens of 2 x 256
// features, 60 us (257 MB: 4.3 TB/s); an 8k bf16 prompt of 8 x 128, e4m3, 25 us
// (50 MB, three quarters of the issue slots); 64 decode tokens 5.9 us.  Indexes of
// compile-time head dimensions and page shifts: 65, 30 and 6.3 us with divisions.
// A thread's places of a group kept across groups took registers (48 for 36) and
// lost (63 and 28 us under the same profile that gives this 62 and 27).
template <int D, bool E4M3, bool BF16>
__global__ void __launch_bounds__(kAppendThreads)
kv8_append_kernel(Kv8Cache c, Kv8Step s, const void *keys, uint64_t k_stride, const void *values, uint64_t v_stride,
                  ErrorWord err) {
    __shared__ uint32_t warp_max[kAppendThreads / 32], warp_rows[kAppendThreads / 32];
    constexpr uint32_t quads = D / 4;
    const uint32_t tid = threadIdx.x, P = c.page_tokens;
    const uint32_t head = blockIdx.y >> 1, side = blockIdx.y & 1u;
    pdl_wait();
    // the slots and the first rows are on their way while the run is looked at
    const int32_t first = s.page_runs[blockIdx.x];
    const uint32_t room = (uint32_t)first < s.tokens ? min(P, s.tokens - (uint32_t)first) : 0u;
    const int64_t slot = room > 0 ? s.slots[first] : -1, mine = tid < room ? s.slots[first + tid] : -1;
    const void *rows = side ? values : keys;
    const uint64_t stride = side ? v_stride : k_stride, base = (uint64_t)first * stride + (uint64_t)head * D;
    float4 ahead[kAhead];
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i) {
        const uint32_t row = (tid + i * kAppendThreads) / quads, f = (tid + i * kAppendThreads) % quads * 4;
        ahead[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (row < room) ahead[i] = load4<BF16>(rows, base + row * stride + f);
    }
    if (__syncthreads_or(first < 0 || (tid == 0 && err_raised(err)))) return;
    if (slot < 0 || slot >= (int64_t)c.pages * P) {   // no room: first is behind the rows
        if (tid == 0) raise(err, kErrStep);
        return;
    }
    const uint32_t page_shift = __ffs(P) - 1;   // a power of two
    const uint64_t page = (uint64_t)slot >> page_shift;
    const uint32_t at = (uint32_t)slot & (P - 1), most = min(P - at, room);
    // the run ends before the first row whose slot does not follow
    const uint32_t other = __ballot_sync(~0u, tid >= most || mine != slot + (int64_t)tid);
    if ((tid & 31) == 0) warp_rows[tid >> 5] = other != 0 ? tid + __ffs(other) - 1 : P;
    __syncthreads();
    uint32_t n = P;
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) n = min(n, warp_rows[w]);
    const uint32_t end = at + n;

    // |x| as integers order like the floats, infinities and NaNs above all
    uint32_t top = 0;
    auto see = [&](float4 x) {
        top = max(max(top, __float_as_uint(x.x) & 0x7fffffffu), __float_as_uint(x.y) & 0x7fffffffu);
        top = max(max(top, __float_as_uint(x.z) & 0x7fffffffu), __float_as_uint(x.w) & 0x7fffffffu);
    };
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i)
        if (tid + i * kAppendThreads < n * quads) see(ahead[i]);
#pragma unroll 4
    for (uint32_t u = tid + kAhead * kAppendThreads; u < n * quads; u += kAppendThreads)
        see(load4<BF16>(rows, base + (uint64_t)(u / quads) * stride + u % quads * 4));
    top = __reduce_max_sync(~0u, top);
    if ((tid & 31) == 0) warp_max[tid >> 5] = top;
    float *scale_at = c.scales + (page * c.heads + head) * 2 + side;
    const float old = at > 0 ? *scale_at : 0.0f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) top = max(top, warp_max[w]);
    if (top >= 0x7f800000u) {   // a non-finite value: this page keeps what it holds
        if (tid == 0) raise(err, kErrNonFinite);
        return;
    }
    const float scale = fmaxf(old, __fdiv_rn(__uint_as_float(top), kLargest<E4M3>));
    const bool grown = at > 0 && scale > old;
    const float ratio = grown ? __fdiv_rn(old, scale) : 1.0f;

    // Groups of 16 tokens that change: all of a page that the run begins
    // (the rows behind it are cleared), those before the run too if the scale
    // grew, else those that the run touches.
    const uint32_t g0 = at == 0 || grown ? 0u : at / 16, g1 = at == 0 ? P / 16 : (end + 15) / 16;
    uint8_t *codes = c.codes + (page * c.heads + head) * (2ull * P * D) + side * 16u * D;
    auto recode = [&](uint32_t byte) {
        return encode<E4M3>(__fmul_rn(decode<E4M3>(byte), ratio));
    };
    auto exact = [&](float x) { return encode<E4M3>(scale > 0.0f ? __fdiv_rn(x, scale) : 0.0f); };
    // the reciprocal's path wants normal numbers
    const bool plain = scale < 1.0e-30f || scale > 1.0e30f;
    const float inv = plain ? 0.0f : __frcp_rn(scale);
    const float low = inv * (1.0f - 0x1p-22f), high = inv * (1.0f + 0x1p-22f);
    auto fresh4 = [&](float4 x) {
        bool near = plain;
        uint32_t w = encode4<E4M3>(x, low, high, near);
        if (near) w = exact(x.x) | exact(x.y) << 8 | exact(x.z) << 16 | exact(x.w) << 24;
        return w;
    };
    for (uint32_t u = g0 * D + tid; u < g1 * D; u += kAppendThreads) {   // D units of 16 bytes in a group
        const uint32_t group = u / D, w = u % D;
        uint4 *unit = reinterpret_cast<uint4 *>(codes + (uint64_t)group * 32 * D + w * 16);
        uint32_t word[4];
        if (side == 0) {
            const uint32_t row = group * 16 + w / 32 % 2 * 8 + w % 32 / 4, f = w / 64 * 64 + w % 4 * 16;
            if (row >= at && row < end) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 x = load4<BF16>(rows, base + (uint64_t)(row - at) * stride + f + 4 * i);
                    word[i] = fresh4(x);
                }
            } else if (at == 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) word[i] = kZeroByte<E4M3> * 0x01010101u;
            } else if (row < at && grown) {
                const uint4 had = *unit;
                const uint32_t h[4] = {had.x, had.y, had.z, had.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    word[i] = 0;
#pragma unroll
                    for (int b = 0; b < 4; ++b) word[i] |= recode(h[i] >> (8 * b) & 0xffu) << (8 * b);
                }
            } else {
                continue;
            }
        } else {
            const uint32_t f = w / 32 * 32 + w % 32 / 4 * 4, t0 = group * 16 + w % 4 * 2;   // tokens t0 + {0, 1, 8, 9}
            if (at > 0) {
                const uint4 had = *unit;
                word[0] = had.x, word[1] = had.y, word[2] = had.z, word[3] = had.w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) word[i] = kZeroByte<E4M3> * 0x01010101u;
            }
            bool changed = at == 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t row = t0 + (k >> 1) * 8 + (k & 1), keep = ~(0xffu << (8 * k));
                if (row >= at && row < end) {
                    const float4 x = load4<BF16>(rows, base + (uint64_t)(row - at) * stride + f);
                    const uint32_t four = fresh4(x);   // one byte of each word
#pragma unroll
                    for (int i = 0; i < 4; ++i)   // byte k of the word becomes byte i of the four
                        word[i] = __byte_perm(word[i], four, (0x3210u & ~(0xfu << (4 * k))) | (4u + i) << (4 * k));
                    changed = true;
                } else if (row < at && grown) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        word[i] = (word[i] & keep) | recode(word[i] >> (8 * k) & 0xffu) << (8 * k);
                    changed = true;
                }
            }
            if (!changed) continue;
        }
        *unit = make_uint4(word[0], word[1], word[2], word[3]);
    }
    if (tid == 0 && (at == 0 || grown)) *scale_at = scale;
}

void launch_kv8_append(const Kv8Cache &c, const Kv8Step &s, const void *k, uint64_t k_stride, const void *v,
                       uint64_t v_stride, uint32_t bf16, ErrorWord err, cudaStream_t stream) {
    KernelTimer timer("kv8_append", stream);
    const dim3 grid(s.runs, 2 * c.heads);
    auto go = [&](auto kernel) { launch_pdl(kernel, grid, kAppendThreads, 0, stream, c, s, k, k_stride, v, v_stride, err); };
    auto typed = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        if (c.e4m3)
            bf16 ? go(kv8_append_kernel<D, true, true>) : go(kv8_append_kernel<D, true, false>);
        else
            bf16 ? go(kv8_append_kernel<D, false, true>) : go(kv8_append_kernel<D, false, false>);
    };
    by_dimension(c.dim, typed);
    count_launch();
}

// ------------------------------------------------------------------- read

namespace {
constexpr int kReadThreads = 256;
constexpr uint32_t kReadUnits = 4;   // of 16 values, per thread
}

// The F32 values code * scale of pages[i], natural order: out
// [i][head][key, value][token][feature].  One CTA per (page, head, side) and
// 16 K values; a thread turns 4 key bytes into 4 features of a token, or 16
// value bytes into 4 features of 4 tokens, so that 128 contiguous bytes or more
// are written together; all its loads are on their way before the first store.
// Bound: HBM (4 bytes written per byte read).  Measured under ncu, caches cold:
// 835 pages of 64 tokens, 2 x 256 features, 47 us for 274 MB (5.8 TB/s); 64 such
// pages 6.7 us (11.7 with a CTA per page side that loads as it goes).  16, 32 and
// 64 values a thread: 61, 51 and 50 us for the 835 pages by events.
template <int D, bool E4M3>
__global__ void __launch_bounds__(kReadThreads)
kv8_read_kernel(Kv8Cache c, const int32_t *__restrict__ pages, float *__restrict__ out, ErrorWord err) {
    const uint32_t P = c.page_tokens, head = blockIdx.y >> 1, side = blockIdx.y & 1u;
    pdl_wait();
    const int32_t page = pages[blockIdx.x];
    if (err_raised(err)) return;
    if (page < 0 || (uint32_t)page >= c.pages) {
        if (threadIdx.x == 0) raise(err, kErrStep);
        return;
    }
    const uint8_t *codes = c.codes + ((uint64_t)page * c.heads + head) * (2ull * P * D) + side * 16u * D;
    const float scale = c.scales[((uint64_t)page * c.heads + head) * 2 + side];
    float *o = out + (((uint64_t)blockIdx.x * c.heads + head) * 2 + side) * P * D;
    if (side == 0) {
        uint32_t b[4 * kReadUnits];
#pragma unroll
        for (uint32_t i = 0; i < 4 * kReadUnits; ++i) {
            const uint32_t u = (blockIdx.z * 4 * kReadUnits + i) * kReadThreads + threadIdx.x;
            const uint32_t row = u / (D / 4), f = u % (D / 4) * 4, w = row % 16;
            if (row < P)
                b[i] = *reinterpret_cast<const uint32_t *>(codes + (uint64_t)(row / 16) * 32 * D + f / 64 * 1024 + w / 8 * 512 +
                                                           w % 8 * 64 + f % 64);
        }
#pragma unroll
        for (uint32_t i = 0; i < 4 * kReadUnits; ++i) {
            const uint32_t u = (blockIdx.z * 4 * kReadUnits + i) * kReadThreads + threadIdx.x;
            if (u < P * D / 4)
                reinterpret_cast<float4 *>(o)[u] =
                    make_float4(__fmul_rn(decode<E4M3>(b[i] & 0xffu), scale), __fmul_rn(decode<E4M3>(b[i] >> 8 & 0xffu), scale),
                                __fmul_rn(decode<E4M3>(b[i] >> 16 & 0xffu), scale), __fmul_rn(decode<E4M3>(b[i] >> 24), scale));
        }
    } else {
        uint4 b[kReadUnits];
#pragma unroll
        for (uint32_t i = 0; i < kReadUnits; ++i) {
            const uint32_t u = (blockIdx.z * kReadUnits + i) * kReadThreads + threadIdx.x;
            if (u < P * D / 16) b[i] = *reinterpret_cast<const uint4 *>(codes + (uint64_t)(u / D) * 32 * D + u % D * 16);
        }
#pragma unroll
        for (uint32_t i = 0; i < kReadUnits; ++i) {
            const uint32_t u = (blockIdx.z * kReadUnits + i) * kReadThreads + threadIdx.x, w = u % D;
            const uint32_t f = w / 32 * 32 + w % 32 / 4 * 4, t0 = u / D * 16 + w % 4 * 2;
            if (u >= P * D / 16) break;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t row = t0 + (k >> 1) * 8 + (k & 1);
                *reinterpret_cast<float4 *>(o + (uint64_t)row * D + f) =
                    make_float4(__fmul_rn(decode<E4M3>(b[i].x >> (8 * k) & 0xffu), scale),
                                __fmul_rn(decode<E4M3>(b[i].y >> (8 * k) & 0xffu), scale),
                                __fmul_rn(decode<E4M3>(b[i].z >> (8 * k) & 0xffu), scale),
                                __fmul_rn(decode<E4M3>(b[i].w >> (8 * k) & 0xffu), scale));
            }
        }
    }
}

void launch_kv8_read(const Kv8Cache &c, const int32_t *pages, uint32_t count, float *out, ErrorWord err,
                     cudaStream_t stream) {
    KernelTimer timer("kv8_read", stream);
    const uint32_t each = 16 * kReadUnits * kReadThreads;   // values of a CTA
    const dim3 grid(count, 2 * c.heads, (c.page_tokens * c.dim + each - 1) / each);
    by_dimension(c.dim, [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        if (c.e4m3)
            launch_pdl(kv8_read_kernel<D, true>, grid, kReadThreads, 0, stream, c, pages, out, err);
        else
            launch_pdl(kv8_read_kernel<D, false>, grid, kReadThreads, 0, stream, c, pages, out, err);
    });
    count_launch();
}

}  // namespace kqb
