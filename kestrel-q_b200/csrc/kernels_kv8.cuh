// Device code that the paged cache's attention kernels share: bounded waits,
// bulk copies, code conversion, requests of a step, finished rows.
#pragma once

#include "kernels_kv8.hpp"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace kqb {

namespace {

constexpr uint32_t kG = kKv8GroupTokens;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kRaise = 8.0f;        // a logit this far above its reference point raises that
constexpr float kWeightBits = 6.0f;
constexpr float kMost = 3.40282347e38f;
constexpr uint32_t kTryNs = 100000;
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr uint32_t kPromptUnit = 8;   // groups: a prompt's split is whole steps of 128 tokens

__device__ __forceinline__ bool err_raised(const ErrorWord &e) {
    return *reinterpret_cast<volatile unsigned long long *>(e.word) != 0ull;
}

__device__ __forceinline__ void raise(const ErrorWord &e, uint32_t code) {
    atomicCAS(e.word, 0ull, ((unsigned long long)code << 32) | e.call_id);
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

__device__ __forceinline__ uint64_t global_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// Bounded wait for the phase of `bar` with the given parity: gives up after
// kWaitNs, or (quit not null) once *quit is set, and sets it then.  Each try
// may suspend the thread for up to kTryNs: a warp that polls takes issue slots
// from the others of its scheduler.
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, volatile uint32_t *quit = nullptr) {
    uint64_t t0 = 0;   // the clock is read only once a wait is slow
#pragma unroll 1
    for (uint32_t i = 0;; ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.b32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(smem_u32(bar)), "r"(parity), "r"(kTryNs)
            : "memory");
        if (done) return true;
        if ((i & 15) == 15) {
            if (quit != nullptr && *quit) return false;
            const uint64_t now = global_ns();
            if (t0 == 0) t0 = now;
            else if (now - t0 > kWaitNs) break;
        }
    }
    if (quit != nullptr) *quit = 1;
    return false;
}

// The same for a whole warp, with the same answer in every lane; one lane
// polls (polls are shared-memory traffic: with all lanes the row kernel took
// 203 us for 64 F32 sequences, not 192).  What that lane's wait acquired is
// ordered before the other lanes' accesses by the warp barrier; a shuffle
// orders no memory.
__device__ __forceinline__ bool bar_wait_warp(uint64_t *bar, uint32_t parity, volatile uint32_t *quit = nullptr) {
    uint32_t ok = 0;
    if ((threadIdx.x & 31) == 0) ok = bar_wait(bar, parity, quit);
    __syncwarp();
    return __shfl_sync(~0u, ok, 0) != 0;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A row's two reference points, whole numbers, so that every factor made of
// them is an exact power of two: m for logits and the sum l, m + z for O, whose
// weights have the page's value scale in them.  A weight enters the second
// product as
//   p sV 2^(6 - z),   p = 2^(l - m)
// at most 2^14; it loses bits only where it is small beside the row's largest
// p sV, however large the values that the row does not attend to.  Either point
// moves when it is 8 below a step's largest.  Scales below 2^-110 count as that:
// z, at most 9 below them, keeps 2^(6 - z) and 2^(z - 6) normal numbers.  A
// page of scale 2^-119 still has 22 bits (weights of 2^-3 and more), one of
// 2^-142 counts as zeros.  sV 2^(6 - z) can overflow only where p is below
// 2^-114 (p sV is 2^(z + 8) at most), and stays finite then.
__device__ __forceinline__ float size_of(float scale) { return fmaxf(__log2f(scale), -110.0f); }
__device__ __forceinline__ float weight_of(float m, float z) {   // of p sV
    return m == -INFINITY ? 0.0f : exp2_approx(kWeightBits - z);
}
__device__ __forceinline__ float back_of(float m, float z) {   // of O, to units of 2^m
    return m == -INFINITY ? 0.0f : exp2_approx(z - kWeightBits);
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

// Four query elements from element `at` on.
template <bool BF16>
__device__ __forceinline__ float4 load4(const void *base, uint64_t at) {
    if constexpr (BF16) {
        const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const __nv_bfloat16 *>(base) + at);
        return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                           __uint_as_float(w.y & 0xffff0000u));
    } else {
        return *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at);
    }
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

// Four features of a row from its sums: the output and, with the first four,
// the log-sum.
template <bool BF16>
__device__ __forceinline__ void finish4(const Kv8Attend &a, const Request &rq, uint32_t G, uint32_t head, uint32_t row,
                                        uint32_t f, uint32_t dim, float m, float l, float4 o, const ErrorWord &err) {
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
    if (!(l < INFINITY) || !(fabsf(o.x) + fabsf(o.y) + fabsf(o.z) + fabsf(o.w) < INFINITY)) raise(err, kErrNonFinite);
    const uint64_t token = rq.first + row / G;
    const uint32_t qh = head * G + row % G;
    store4<BF16>(a.out, token * a.out_stride + (uint64_t)qh * dim + f, o);
    if (a.lse != nullptr && f == 0) a.lse[token * a.query_heads + qh] = l > 0.0f ? (m + log2f(l)) * kLn2 : -INFINITY;
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

}  // namespace kqb
