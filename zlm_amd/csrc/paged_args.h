// paged_args.h -- the argument blocks of the paged-cache kernels (zlm_paged.hip),
// shared with the host library that fills them.
#pragma once
#include <stdint.h>

namespace zlm {

constexpr uint32_t kPagedMaxSeqs = 1024;  // sequences of one call (their prefix sums live in LDS)

// What every kernel takes of the cache and the batch.  `table` entries are page
// numbers; one outside [0, n_pages) names no page.
struct Paged {
    uint8_t* k;
    uint8_t* v;
    const int32_t* q_start;  // n_seqs + 1: the rows of sequence s are [q_start[s], q_start[s + 1])
    const int32_t* kv_len;   // n_seqs: positions of s including these rows
    const int32_t* table;    // n_seqs x table_stride
    uint32_t n_seqs, n_tokens, table_stride, n_pages;
    uint32_t n_kv, page_shift;
};

struct PagedAppend {
    Paged p;
    const float* qkv;
    const float* q_norm;  // null: no head norm
    const float* k_norm;
    float* q_out;
    uint64_t stride;  // floats between rows of qkv
    uint32_t n_heads;
    uint32_t per;     // heads a wave takes at a time: 1 or 4
    float eps;
    double log_base;  // of the rotation's base
};

struct PagedRead {
    Paged p;
    float* k_out;
    float* v_out;
};

struct PagedAttend {
    Paged p;
    const float* q;
    float* out;
    float* part;       // the shares' partial results
    uint32_t* counts;  // a counter for every share, 0 between calls
    uint32_t n_heads, group;
    uint32_t window;  // 0: all
    float scale;      // times log2(e)
    uint32_t few_rows;  // sequences with more rows (tokens x group) are the many-row kernel's
    uint32_t splits;    // its splits of the positions
};

}  // namespace zlm
