// Internal interface between the host API of rotary positions, pages and chosen pages (abq_decoding.hip) and their kernels
// (abq_rotary.hip, abq_pages.hip, abq_attn_choose.hip, abq_attn_tree.hip).
#pragma once
#include "abq_attn.h"

namespace abq {

// What is turned: rows of queries and keys (heads of 0: none), and where it goes.  cache NULL: only that.
struct RotaryCall {
    abq_rotary rotary;
    abq_rows q, q_out, k, k_out, v; // k_out without data: the turned keys are not kept
    int heads[2], head_dim, dtype;
    int64_t tokens;
    const int32_t *positions;
    int64_t position_stride;
    const abq_kv_cache *cache;
    const int32_t *slots;
};
int rotary_splits(int64_t tokens, int steps);
hipError_t launch_rotary(const RotaryCall &call, hipStream_t stream);

hipError_t launch_pages_fork(const abq_kv_pages &p, const int32_t *parents, hipStream_t stream);
hipError_t launch_pages_extend(const abq_kv_pages &p, const int32_t *counts, int32_t *slots, int64_t rows, int32_t *starts, int32_t *granted, int32_t *copies,
                               hipStream_t stream);
hipError_t launch_pages_compact(const abq_kv_pages &p, int32_t *moves, hipStream_t stream);
hipError_t launch_copy_pages(const abq_kv_cache &c, const abq_kv_bounds *bounds, const int32_t *pairs, int64_t count, hipStream_t stream);

struct ChooseCall {
    abq_kv_cache cache;
    abq_kv_bounds bounds;
    abq_rows q;
    int dtype, heads;
    const int32_t *page_table, *context, *q_starts;
    int max_pages, seqs, max_q, first, last, count;
    int likely; // pages of a sequence, as far as the host knows
    int32_t *blocks;
    void *workspace;
    size_t workspace_bytes;
};
// Bytes of all pages' scores where they are worth a launch of their own; 0 otherwise
size_t choose_workspace_bytes(int seqs, int max_q, int kv_heads, int max_pages, int likely);
int bound_slots(const abq_kv_cache &c, int64_t count); // that a workgroup looks through
hipError_t launch_kv_bound(const abq_kv_cache &c, const abq_kv_bounds &bounds, const int32_t *slots, int64_t count, hipStream_t stream);
hipError_t launch_attn_choose(const ChooseCall &call, hipStream_t stream);

void plan_attn_sparse(abq_sparse_state *st, int most_parts);
hipError_t launch_attn_sparse(const abq_sparse_state &st, hipStream_t stream);

constexpr int kMostSeqs = 8192;      // of a table of pages: what a workgroup scans at once
constexpr int kMostChosen = 32768;   // pages of a sequence that a workgroup keeps the scores of, in 128 KB of LDS

} // namespace abq
