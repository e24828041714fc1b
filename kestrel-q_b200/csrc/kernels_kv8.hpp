// Launch interface of the paged 8-bit key/value cache (kernels_kv8.cu,
// kernels_kv8_attend.cu).
#pragma once

#include "kernels.hpp"

namespace kqb {

constexpr uint32_t kKv8GroupTokens = 16;    // tokens of a group: the unit of the page layout
constexpr uint32_t kKv8MaxRequests = 16384; // plan keeps three prefix sums of every request in shared memory

// Device view of a cache (kq_b200_kv8_cache).  Page p, head h: 2 * P * d
// bytes at ((p * heads + h) * 2 * P * d), P / 16 groups of 32 * d bytes, each
// 16 * d key codes, then 16 * d value codes in the order the attention's
// tensor-core fragments read them:
//   key    [j d/64][h 2][g 8][t 4][e 16]       feature = 64 j + 16 t + e, token = 8 h + g
//   value  [j d/32][g 8][t 4][i 4][h 2][e 2]   feature = 32 j + 4 g + i, token = 8 h + 2 t + e
// int8 codes are stored with 128 added.  scales: [page][head][key, value].
struct Kv8Cache {
    uint8_t *codes;
    float *scales;
    uint32_t heads, dim, page_tokens, pages;
    uint32_t e4m3;   // 0: int8, 1: e4m3
};

// Device view of a step (kq_b200_kv8_step).
struct Kv8Step {
    uint32_t requests, tokens, columns, runs;
    uint64_t table_stride;
    int32_t *table, *query_offsets, *kv_lengths, *positions, *run_offsets, *page_runs;
    int64_t *slots;
};

struct Kv8Plan {
    const int32_t *context, *fresh, *free_pages, *free_head;
    int32_t *free_head_out;
    uint32_t free_count;
};

struct Kv8Attend {
    const void *q;
    void *out;
    float *lse;            // may be null
    uint64_t q_stride, out_stride;   // elements between tokens
    uint32_t query_heads;
    uint32_t bf16;         // query and output type
    float scale_log2;      // softmax scale * log2(e)
    float *workspace;      // partial results of split tiles
};

// How a call's tiles are cut (kv8_attend_shape): by the sizes the host knows.
struct Kv8Shape {
    uint32_t row_tile;      // rows per tile of the row kernel: 8 or 16
    uint32_t row_limit;     // requests of more rows go to the prompt kernel (UINT32_MAX: none do)
    uint32_t row_shares;    // CTAs of the row kernel
    uint32_t join_tiles;    // cut tiles at most, joined by a CTA per 64 features of a row (0: by a CTA per share)
    uint32_t prompt_rows;   // rows per tile of the prompt kernel
    uint32_t prompt_tiles;  // 0: the prompt kernel does not run
    uint32_t prompt_groups, prompt_splits;
    uint64_t row_floats, prompt_floats;   // workspace
};

Kv8Shape kv8_attend_shape(const Kv8Cache &c, const Kv8Step &s, uint32_t query_heads, bool bf16,
                          uint64_t max_kv_length);
uint32_t kv8_prompt_rows(uint32_t dim, bool bf16);

void launch_kv8_plan(const Kv8Cache &c, const Kv8Step &s, const Kv8Plan &p, ErrorWord err, cudaStream_t stream);
void launch_kv8_append(const Kv8Cache &c, const Kv8Step &s, const void *k, uint64_t k_stride, const void *v,
                       uint64_t v_stride, uint32_t bf16, ErrorWord err, cudaStream_t stream);
void launch_kv8_read(const Kv8Cache &c, const int32_t *pages, uint32_t count, float *out, ErrorWord err,
                     cudaStream_t stream);
void launch_kv8_prompt(const Kv8Cache &c, const Kv8Step &s, const Kv8Attend &a, const Kv8Shape &shape, ErrorWord err,
                       cudaStream_t stream);
void launch_kv8_attend(const Kv8Cache &c, const Kv8Step &s, const Kv8Attend &a, const Kv8Shape &shape, ErrorWord err,
                       cudaStream_t stream);

}  // namespace kqb
