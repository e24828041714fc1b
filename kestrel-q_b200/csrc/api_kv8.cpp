// C ABI of the paged 8-bit key/value cache (group 4 of kq_b200.h): checks of
// the arguments the host can see, then one launch sequence on the library
// stream.  The arrays' contents are checked by the kernels.
#include "kernels_kv8.hpp"
#include "runtime.hpp"

#include <algorithm>
#include <cmath>

#include "kq_b200.h"

using namespace kqb;

namespace {

bool geometry_ok(const kq_b200_kv8_cache *c) {
    if (c == nullptr) return false;
    const uint32_t d = c->head_dimension, p = c->page_tokens;
    return c->kv_head_count >= 1 && c->kv_head_count <= 1024 && (d == 64 || d == 128 || d == 256) &&
           (p == 16 || p == 32 || p == 64 || p == 128) && c->page_count >= 1 && c->page_count <= INT32_MAX &&
           (c->format == KQ_B200_KV8_INT8 || c->format == KQ_B200_KV8_E4M3);
}

// Device memory (or managed memory) that kernels on `device` can use.
bool on_device(const void *p, int device) {
    cudaPointerAttributes attr;
    if (p == nullptr || cudaPointerGetAttributes(&attr, p) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    return (attr.type == cudaMemoryTypeDevice && attr.device == device) || attr.type == cudaMemoryTypeManaged;
}

bool aligned(const void *p, uint64_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

struct Span {
    const void *p;
    uint64_t bytes;
};

template <size_t N>
bool any_missing(const Span (&spans)[N]) {
    for (const Span &s : spans)
        if (s.p == nullptr && s.bytes > 0) return true;
    return false;
}

// Every array holds values of 4 bytes or more (what needs more alignment is
// checked where it is known).
template <size_t N>
bool any_misaligned(const Span (&spans)[N]) {
    for (const Span &s : spans)
        if (!aligned(s.p, 4)) return true;
    return false;
}

template <size_t N, size_t M>
bool any_overlap(const Span (&writes)[N], const Span (&reads)[M]) {
    for (size_t i = 0; i < N; ++i) {
        for (const Span &r : reads)
            if (ranges_overlap(writes[i].p, writes[i].bytes, r.p, r.bytes)) return true;
        for (size_t j = i + 1; j < N; ++j)
            if (ranges_overlap(writes[i].p, writes[i].bytes, writes[j].p, writes[j].bytes)) return true;
    }
    return false;
}

// What every call checks of the cache (`with_arrays`: of its arrays too).
kq_status check_cache(const kq_b200_kv8_cache *c, bool with_arrays, Kv8Cache *out, kq_diagnostic *d) {
    if (!geometry_ok(c))
        return fail(d, KQ_STATUS_DIMENSION_MISMATCH,
                    "a cache of 1..1024 heads, head dimension 64, 128 or 256, pages of 16, 32, 64 or 128 tokens and a "
                    "known format is required");
    if (with_arrays) {
        if (c->codes == nullptr || c->scales == nullptr)
            return fail(d, KQ_STATUS_INVALID_ARGUMENT, "cache arrays are required");
        if (c->codes_bytes < kq_b200_kv8_codes_bytes(c) || c->scales_count < kq_b200_kv8_scales_count(c))
            return fail(d, KQ_STATUS_BUFFER_TOO_SMALL, "cache arrays are smaller than its pages");
        if (!aligned(c->codes, 16) || !aligned(c->scales, 8))
            return fail(d, KQ_STATUS_INVALID_ALIGNMENT, "codes need 16-byte, scales 8-byte alignment");
    }
    out->codes = static_cast<uint8_t *>(c->codes);
    out->scales = c->scales;
    out->heads = c->kv_head_count;
    out->dim = c->head_dimension;
    out->page_tokens = c->page_tokens;
    out->pages = c->page_count;
    out->e4m3 = c->format == KQ_B200_KV8_E4M3;
    return KQ_STATUS_OK;
}

// The context of the current device, if every span that is not empty is its
// memory.
template <size_t N, size_t M>
kq_status device_context(const Span (&writes)[N], const Span (&reads)[M], DeviceContext **out, kq_diagnostic *d) {
    const kq_status st = context(out, d);
    if (st != KQ_STATUS_OK) return st;
    for (const Span &w : writes)
        if (w.bytes > 0 && !on_device(w.p, (*out)->device))
            return fail(d, KQ_STATUS_INVALID_ARGUMENT, "an output is not memory of the current device");
    for (const Span &r : reads)
        if (r.bytes > 0 && !on_device(r.p, (*out)->device))
            return fail(d, KQ_STATUS_INVALID_ARGUMENT, "an input is not memory of the current device");
    return KQ_STATUS_OK;
}

kq_status check_step(const kq_b200_kv8_step *s, Kv8Step *out, kq_diagnostic *d) {
    if (s == nullptr || s->request_count == 0 || s->token_capacity == 0 || s->table_columns == 0)
        return fail(d, KQ_STATUS_INVALID_ARGUMENT, "a step with requests, tokens and table columns is required");
    if (s->request_count > kKv8MaxRequests || s->token_capacity > INT32_MAX || s->run_capacity > INT32_MAX)
        return fail(d, KQ_STATUS_LIMIT_EXCEEDED, "a step has at most 16384 requests and 2^31 - 1 tokens");
    if (s->table_stride < s->table_columns)
        return fail(d, KQ_STATUS_DIMENSION_MISMATCH, "block table stride is below its columns");
    if (s->table_stride > (uint64_t)INT64_MAX / 4 / s->request_count)
        return fail(d, KQ_STATUS_ARITHMETIC_OVERFLOW, "block table overflows the address space");
    out->requests = s->request_count;
    out->tokens = s->token_capacity;
    out->columns = s->table_columns;
    out->runs = s->run_capacity;
    out->table_stride = s->table_stride;
    out->table = s->block_table;
    out->query_offsets = s->query_offsets;
    out->kv_lengths = s->kv_lengths;
    out->positions = s->positions;
    out->run_offsets = s->run_offsets;
    out->page_runs = s->page_runs;
    out->slots = s->slots;
    return KQ_STATUS_OK;
}

uint64_t table_bytes(const Kv8Step &s) { return ((uint64_t)(s.requests - 1) * s.table_stride + s.columns) * 4; }

bool known_dtype(kq_b200_kv8_dtype t) { return t == KQ_B200_KV8_F32 || t == KQ_B200_KV8_BF16; }

// Rows [tokens][heads][d] with a token stride in elements: its bytes, or an
// error for a stride that overlaps rows or an unaligned row.
kq_status row_bytes(uint32_t tokens, uint64_t stride, uint64_t width, uint32_t size, const void *p, const char *what,
                    uint64_t *bytes, kq_diagnostic *d) {
    if (stride < width) {
        diag_set(d, KQ_STATUS_DIMENSION_MISMATCH, "%s stride is below a token's elements", what);
        return KQ_STATUS_DIMENSION_MISMATCH;
    }
    uint64_t step, n;
    if (!mul_ok(stride, size, &step) || !mul_ok(tokens - 1, step, &n) || !add_ok(n, width * size, &n) || n > INT64_MAX) {
        diag_set(d, KQ_STATUS_ARITHMETIC_OVERFLOW, "%s rows overflow the address space", what);
        return KQ_STATUS_ARITHMETIC_OVERFLOW;
    }
    if (!aligned(p, 16) || step % 16 != 0) {
        diag_set(d, KQ_STATUS_INVALID_ALIGNMENT, "%s rows must be 16-byte aligned", what);
        return KQ_STATUS_INVALID_ALIGNMENT;
    }
    *bytes = n;
    return KQ_STATUS_OK;
}

// Query heads against the cache, and the launch sizes; `shape` cuts the work.
kq_status check_attend(const Kv8Cache &c, const Kv8Step &s, uint32_t query_heads, bool bf16, uint64_t max_kv_length,
                       Kv8Shape *shape, kq_diagnostic *d) {
    if (query_heads == 0 || query_heads % c.heads != 0)
        return fail(d, KQ_STATUS_DIMENSION_MISMATCH, "query heads must be a multiple of the key/value heads");
    if ((uint64_t)s.tokens * (query_heads / c.heads) > INT32_MAX)
        return fail(d, KQ_STATUS_LIMIT_EXCEEDED, "a step has at most 2^31 - 1 query rows per key/value head");
    *shape = kv8_attend_shape(c, s, query_heads, bf16, max_kv_length);
    const uint64_t prompt = (uint64_t)shape->prompt_tiles * c.heads *
                            std::max<uint64_t>(shape->prompt_splits, shape->prompt_rows);
    if (prompt > INT32_MAX)
        return fail(d, KQ_STATUS_LIMIT_EXCEEDED, "the step is too large for one launch");
    return KQ_STATUS_OK;
}

}  // namespace

extern "C" {

uint64_t kq_b200_kv8_codes_bytes(const kq_b200_kv8_cache *cache) {
    // at most 2^31 pages of 1024 heads * 2 * 128 tokens * 256 bytes: 2^57
    if (!geometry_ok(cache)) return 0;
    return 2ull * cache->page_count * cache->kv_head_count * cache->page_tokens * cache->head_dimension;
}

uint64_t kq_b200_kv8_scales_count(const kq_b200_kv8_cache *cache) {
    return geometry_ok(cache) ? 2ull * cache->page_count * cache->kv_head_count : 0;
}

uint64_t kq_b200_kv8_run_capacity(uint32_t tokens, uint32_t requests, uint32_t page_tokens) {
    if (page_tokens == 0) return 0;
    return std::min<uint64_t>(tokens, tokens / page_tokens + 2ull * requests);
}

kq_status kq_b200_kv8_plan(const kq_b200_kv8_cache *cache, const kq_b200_kv8_step *step, const int32_t *context_lengths,
                           const int32_t *new_lengths, const int32_t *free_pages, uint32_t free_count,
                           const int32_t *free_head, int32_t *free_head_out, kq_diagnostic *diagnostic) {
    kq_diagnostic_clear(diagnostic);
    Kv8Cache c;
    Kv8Step s;
    kq_status st = check_cache(cache, false, &c, diagnostic);
    if (st == KQ_STATUS_OK) st = check_step(step, &s, diagnostic);
    if (st != KQ_STATUS_OK) return st;
    if (free_count > INT32_MAX) return fail(diagnostic, KQ_STATUS_LIMIT_EXCEEDED, "at most 2^31 - 1 free pages");
    const uint64_t B = s.requests;
    const Span writes[] = {{s.table, table_bytes(s)}, {s.query_offsets, 4 * (B + 1)}, {s.kv_lengths, 4 * B},
                           {s.slots, 8ull * s.tokens}, {s.positions, 4ull * s.tokens}, {s.run_offsets, 4 * (B + 1)},
                           {s.page_runs, 4ull * s.runs}, {free_head_out, 4}};
    const Span reads[] = {{context_lengths, 4 * B}, {new_lengths, 4 * B}, {free_pages, 4ull * free_count}, {free_head, 4}};
    if (s.runs == 0 || any_missing(writes) || any_missing(reads))
        return fail(diagnostic, KQ_STATUS_INVALID_ARGUMENT, "a plan takes lengths, a free list and every array of the step");
    if (!aligned(s.slots, 8)) return fail(diagnostic, KQ_STATUS_INVALID_ALIGNMENT, "slots need 8-byte alignment");
    if (any_misaligned(writes) || any_misaligned(reads))
        return fail(diagnostic, KQ_STATUS_INVALID_ALIGNMENT, "arrays need 4-byte alignment");
    if (any_overlap(writes, reads))
        return fail(diagnostic, KQ_STATUS_ALIASING_VIOLATION, "a plan's outputs must not overlap each other or its inputs");
    DeviceContext *ctx;
    st = device_context(writes, reads, &ctx, diagnostic);
    if (st != KQ_STATUS_OK) return st;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    const Kv8Plan p{context_lengths, new_lengths, free_pages, free_head, free_head_out, free_count};
    launch_kv8_plan(c, s, p, ctx->begin_call(), ctx->stream);
    KQB_CUDA(cudaGetLastError(), diagnostic, "cache plan launch");
    return KQ_STATUS_OK;
}

kq_status kq_b200_kv8_append(const kq_b200_kv8_cache *cache, const kq_b200_kv8_step *step, kq_b200_kv8_dtype dtype,
                             const void *key, uint64_t key_stride, const void *value, uint64_t value_stride,
                             kq_diagnostic *diagnostic) {
    kq_diagnostic_clear(diagnostic);
    Kv8Cache c;
    Kv8Step s;
    kq_status st = check_cache(cache, true, &c, diagnostic);
    if (st == KQ_STATUS_OK) st = check_step(step, &s, diagnostic);
    if (st != KQ_STATUS_OK) return st;
    if (!known_dtype(dtype)) return fail(diagnostic, KQ_STATUS_UNSUPPORTED_TENSOR_TYPE, "rows are F32 or BF16");
    const uint32_t size = dtype == KQ_B200_KV8_F32 ? 4 : 2;
    const uint64_t width = (uint64_t)c.heads * c.dim;
    uint64_t kb, vb;
    st = row_bytes(s.tokens, key_stride, width, size, key, "key", &kb, diagnostic);
    if (st == KQ_STATUS_OK) st = row_bytes(s.tokens, value_stride, width, size, value, "value", &vb, diagnostic);
    if (st != KQ_STATUS_OK) return st;
    const Span writes[] = {{c.codes, kq_b200_kv8_codes_bytes(cache)}, {c.scales, 4 * kq_b200_kv8_scales_count(cache)}};
    const Span reads[] = {{key, kb}, {value, vb}, {s.slots, 8ull * s.tokens}, {s.page_runs, 4ull * s.runs}};
    if (s.runs == 0 || any_missing(reads))
        return fail(diagnostic, KQ_STATUS_INVALID_ARGUMENT, "an append takes key and value rows, slots and page runs");
    if (!aligned(s.slots, 8)) return fail(diagnostic, KQ_STATUS_INVALID_ALIGNMENT, "slots need 8-byte alignment");
    if (any_misaligned(writes) || any_misaligned(reads))
        return fail(diagnostic, KQ_STATUS_INVALID_ALIGNMENT, "arrays need 4-byte alignment");
    if (any_overlap(writes, reads))
        return fail(diagnostic, KQ_STATUS_ALIASING_VIOLATION, "cache arrays must not overlap each other or the rows");
    DeviceContext *ctx;
    st = device_context(writes, reads, &ctx, diagnostic);
    if (st != KQ_STATUS_OK) return st;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    launch_kv8_append(c, s, key, key_stride, value, value_stride, dtype == KQ_B200_KV8_BF16, ctx->begin_call(), ctx->stream);
    KQB_CUDA(cudaGetLastError(), diagnostic, "cache append launch");
    return KQ_STATUS_OK;
}

kq_status kq_b200_kv8_read(const kq_b200_kv8_cache *cache, const int32_t *pages, uint32_t count, float *values,
                           uint64_t values_capacity, kq_diagnostic *diagnostic) {
    kq_diagnostic_clear(diagnostic);
    Kv8Cache c;
    kq_status st = check_cache(cache, true, &c, diagnostic);
    if (st != KQ_STATUS_OK) return st;
    if (count == 0 || count > INT32_MAX || pages == nullptr || values == nullptr)
        return fail(diagnostic, KQ_STATUS_INVALID_ARGUMENT, "page ids and room for their values are required");
    uint64_t want;
    if (!mul_ok(2ull * c.heads * c.page_tokens * c.dim, count, &want) || want > values_capacity || want > INT64_MAX / 4)
        return fail(diagnostic, KQ_STATUS_BUFFER_TOO_SMALL, "values are smaller than the pages");
    if (!aligned(values, 16)) return fail(diagnostic, KQ_STATUS_INVALID_ALIGNMENT, "values need 16-byte alignment");
    const Span writes[] = {{values, want * 4}};
    const Span reads[] = {{c.codes, kq_b200_kv8_codes_bytes(cache)}, {c.scales, 4 * kq_b200_kv8_scales_count(cache)},
                          {pages, 4ull * count}};
    if (any_misaligned(writes) || any_misaligned(reads))
        return fail(diagnostic, KQ_STATUS_INVALID_ALIGNMENT, "arrays need 4-byte alignment");
    if (any_overlap(writes, reads))
        return fail(diagnostic, KQ_STATUS_ALIASING_VIOLATION, "values must not overlap the cache or the page ids");
    DeviceContext *ctx;
    st = device_context(writes, reads, &ctx, diagnostic);
    if (st != KQ_STATUS_OK) return st;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    launch_kv8_read(c, pages, count, values, ctx->begin_call(), ctx->stream);
    KQB_CUDA(cudaGetLastError(), diagnostic, "cache read launch");
    return KQ_STATUS_OK;
}

kq_status kq_b200_kv8_attend_workspace_bytes(const kq_b200_kv8_cache *cache, const kq_b200_kv8_step *step,
                                             uint32_t query_heads, uint64_t max_kv_length, uint64_t *bytes,
                                             kq_diagnostic *diagnostic) {
    kq_diagnostic_clear(diagnostic);
    if (bytes == nullptr) return fail(diagnostic, KQ_STATUS_INVALID_ARGUMENT, "a result is required");
    Kv8Cache c;
    Kv8Step s;
    Kv8Shape shape{};
    kq_status st = check_cache(cache, false, &c, diagnostic);
    if (st == KQ_STATUS_OK) st = check_step(step, &s, diagnostic);
    uint64_t most = 0;
    for (int bf16 = 0; bf16 < 2 && st == KQ_STATUS_OK; ++bf16) {   // enough for either type
        st = check_attend(c, s, query_heads, bf16 != 0, max_kv_length, &shape, diagnostic);
        most = std::max(most, 4 * (shape.row_floats + shape.prompt_floats));
    }
    if (st == KQ_STATUS_OK) *bytes = most;
    return st;
}

kq_status kq_b200_kv8_attend(const kq_b200_kv8_cache *cache, const kq_b200_kv8_step *step, kq_b200_kv8_dtype dtype,
                             const void *query, uint64_t query_stride, uint32_t query_heads, float softmax_scale,
                             uint64_t max_kv_length, void *output, uint64_t output_stride, float *lse, void *workspace,
                             uint64_t workspace_bytes, kq_diagnostic *diagnostic) {
    kq_diagnostic_clear(diagnostic);
    Kv8Cache c;
    Kv8Step s;
    Kv8Shape shape;
    kq_status st = check_cache(cache, true, &c, diagnostic);
    if (st == KQ_STATUS_OK) st = check_step(step, &s, diagnostic);
    if (st == KQ_STATUS_OK)
        st = check_attend(c, s, query_heads, dtype == KQ_B200_KV8_BF16, max_kv_length, &shape, diagnostic);
    if (st != KQ_STATUS_OK) return st;
    if (!known_dtype(dtype)) return fail(diagnostic, KQ_STATUS_UNSUPPORTED_TENSOR_TYPE, "queries are F32 or BF16");
    const float scale_log2 = softmax_scale * 1.44269504088896340736f;
    if (!std::isfinite(scale_log2)) return fail(diagnostic, KQ_STATUS_INVALID_ARGUMENT, "softmax scale must be finite");
    const uint32_t size = dtype == KQ_B200_KV8_F32 ? 4 : 2;
    const uint64_t width = (uint64_t)query_heads * c.dim, B = s.requests;
    uint64_t qb, ob;
    st = row_bytes(s.tokens, query_stride, width, size, query, "query", &qb, diagnostic);
    if (st == KQ_STATUS_OK) st = row_bytes(s.tokens, output_stride, width, size, output, "output", &ob, diagnostic);
    if (st != KQ_STATUS_OK) return st;
    const uint64_t need = 4 * (shape.row_floats + shape.prompt_floats);
    if (workspace_bytes < need || (need > 0 && workspace == nullptr))
        return fail(diagnostic, KQ_STATUS_BUFFER_TOO_SMALL, "attention work space is too small");
    if (need > 0 && !aligned(workspace, 16))
        return fail(diagnostic, KQ_STATUS_INVALID_ALIGNMENT, "work space needs 16-byte alignment");
    const Span writes[] = {{output, ob}, {lse, lse ? 4ull * s.tokens * query_heads : 0}, {workspace, need}};
    const Span reads[] = {{query, qb}, {c.codes, kq_b200_kv8_codes_bytes(cache)},
                          {c.scales, 4 * kq_b200_kv8_scales_count(cache)}, {s.table, table_bytes(s)},
                          {s.query_offsets, 4 * (B + 1)}, {s.kv_lengths, 4 * B}};
    if (any_missing(writes) || any_missing(reads))
        return fail(diagnostic, KQ_STATUS_INVALID_ARGUMENT,
                    "attention takes queries, an output, a block table, query offsets and lengths");
    if (any_misaligned(writes) || any_misaligned(reads))
        return fail(diagnostic, KQ_STATUS_INVALID_ALIGNMENT, "arrays need 4-byte alignment");
    if (any_overlap(writes, reads))
        return fail(diagnostic, KQ_STATUS_ALIASING_VIOLATION, "attention outputs must not overlap each other or its inputs");
    DeviceContext *ctx;
    st = device_context(writes, reads, &ctx, diagnostic);
    if (st != KQ_STATUS_OK) return st;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    const Kv8Attend a{query, output, lse, query_stride, output_stride, query_heads, dtype == KQ_B200_KV8_BF16,
                      scale_log2, static_cast<float *>(workspace)};
    launch_kv8_attend(c, s, a, shape, ctx->begin_call(), ctx->stream);
    KQB_CUDA(cudaGetLastError(), diagnostic, "cache attention launch");
    return KQ_STATUS_OK;
}

}  // extern "C"
