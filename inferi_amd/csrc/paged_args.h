// Kernel argument blocks of the paged-cache operators (device/paged.h,
// device/paged_attn.h), laid out the same on the host and the device.
#pragma once
#include <stdint.h>

namespace ifr {

constexpr uint32_t PG_RELEASE = 0xFFFFFFFFu; // IFR_RELEASE
constexpr uint32_t PG_NO_ROW = 0xFFFFFFFFu;  // IFR_NO_ROW
constexpr uint32_t PG_PLAN_THREADS = 1024;   // requests of one round of paged_plan_k
constexpr uint32_t PG_ROPE_THREADS = 256;

struct PagedPlanArgs {
    const uint32_t *ctx_len, *new_len;
    uint32_t *free_pages;
    const uint32_t *free_count;
    uint32_t *free_count_out, *table, *ctx_len_out, *row_start, *kv_len, *positions;
    uint64_t *slots;
    uint32_t n_requests, n_rows, n_pages, lp, max_pages; // page size 1 << lp
    uint32_t rows_here; // the plan kernel fills the rows and the table itself
    uint32_t *pops;     // else: where each request's popped pages begin; after the last, the stack's height
};

struct PagedRopeArgs {
    const float *q, *k, *v;
    const uint32_t *positions;
    const uint64_t *slots;
    void *q_out, *key, *value;
    int64_t ld_q, ld_k, ld_v, ld_q_out, page_stride, row_stride, head_stride;
    double log2_base;
    uint32_t n_rows, n_heads, n_kv, hs, n_pages, lp;
    uint32_t neox, turn, q_f16, kv_f16;
    uint32_t parts; // workgroups that share a row
};

struct PagedAttnArgs {
    const void *q, *key, *value;
    void *out;
    const uint32_t *table, *row_start, *kv_len;
    float *part_o, *part_ml; // [row][head][split][hs], [row][head][split][2]
    int64_t ld_q, ld_out, page_stride, row_stride, head_stride;
    uint32_t n_pages, lp, max_pages, n_kv, hs, G, n_requests, n_rows;
    uint32_t window, sinks; // window 0: none
    uint32_t n_splits, chunk; // workgroups that share a tile's keys, at most; key tiles of each, at least
    uint32_t QT, heads_per, n_sub; // queries of a tile; heads of a sub-group; sub-groups of a KV head's heads
    uint32_t search; // a workgroup finds its tile among all requests' (else: tile = request)
    uint32_t sorted; // the longest tiles or splits of up to 64 requests first
    float scale2;                  // scale x log2(e)
};

} // namespace ifr
