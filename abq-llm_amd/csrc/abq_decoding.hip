// Host side of what include/abq_attention.h declares around attention: rotary positions, pages of sequences, attention to chosen
// pages.  Argument checks and sizes; no entry point allocates device or host memory.
#include "abq_decoding.h"

#include <string.h>

#include "abq_attn_checks.h"

namespace abq {

namespace {

constexpr int kSparseKind = 3;

bool aligned(const void *p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
bool dtype_valid(int dtype) { return dtype == ABQ_F16 || dtype == ABQ_BF16; }

abq_status check_rotary(const abq_rotary *r, int head_dim, const int32_t *positions, int64_t stride, int64_t rows)
{
    if (!r || !r->turns || !aligned(r->turns, 8) || (rows && !positions) || r->rotary_dim <= 0 || r->rotary_dim % 16 || r->rotary_dim > head_dim || r->axes < 1 ||
        r->axes > 8 || stride < 0 || (r->axes > 1 && stride < rows))
        return ABQ_ERR_INVALID_ARG;
    return ABQ_OK;
}

// Rows that are turned, and where they go: the same ones, or others
abq_status check_turned(const abq_rows *in, const abq_rows *out, int64_t rows, int heads, int head_dim)
{
    abq_status s;
    if (heads <= 0)
        return ABQ_ERR_INVALID_ARG;
    if ((s = check_rows(in, rows, heads, head_dim)) != ABQ_OK || (s = check_rows(out, rows, heads, head_dim, true)) != ABQ_OK)
        return s;
    if (rows && in->data == out->data && ((rows > 1 && in->row_stride != out->row_stride) || (heads > 1 && in->head_stride != out->head_stride)))
        return ABQ_ERR_INVALID_ARG;
    return ABQ_OK;
}

// Whether results begin where other rows do, which other waves read or write: these lie on one another, whatever their strides
bool begins_on(const abq_rows *out, const abq_rows *other) { return out && other && out->rows > 0 && out->data == other->data; }
bool crossed(const abq_rows *q, const abq_rows *q_out, const abq_rows *k, const abq_rows *k_out)
{
    return begins_on(q_out, k) || begins_on(q_out, k_out) || begins_on(k_out, q);
}

// Workgroups of a launch that turns rows of these heads (and of one that quantises values beside it)
abq_status check_turning(const RotaryCall &c, int64_t further)
{
    const int rows = 64 / (c.head_dim / 16);
    if (c.tokens > 0x7ffffff0 || product(c.heads[0], c.head_dim, 1) > 0x7fffffff || product(c.heads[1], c.head_dim, 1) > 0x7fffffff)
        return ABQ_ERR_TOO_LARGE;
    const int steps = (int)(((int64_t)c.heads[0] + rows - 1) / rows + ((int64_t)c.heads[1] + rows - 1) / rows);
    return (product(c.tokens, rotary_splits(c.tokens, steps), 1) + 3) / 4 + further > kMostBlocks ? ABQ_ERR_TOO_LARGE : ABQ_OK;
}

abq_status check_pages(const abq_kv_pages *p)
{
    if (!p || p->seqs <= 0 || p->max_pages <= 0 || p->num_pages <= 0 || p->page_size < 16 || p->page_size > 4096 || (p->page_size & (p->page_size - 1)) ||
        (int64_t)p->num_pages * p->page_size > 0x7fffffff || !p->table || !p->lengths || !p->refs)
        return ABQ_ERR_INVALID_ARG;
    // (workgroups of 1024 threads for two columns each, or more, and one)
    if (p->seqs > kMostSeqs || (int64_t)p->max_pages * p->page_size > 0x7fffffff - 64 || p->max_pages > kMostThreads / 1024 - 2)
        return ABQ_ERR_TOO_LARGE;
    return ABQ_OK;
}

abq_status check_bounds(const abq_kv_bounds *b)
{
    return b && b->codes && b->scales && aligned16(b->codes) && aligned(b->scales, 4) ? ABQ_OK : ABQ_ERR_INVALID_ARG;
}

int likely_pages(const abq_kv_cache *c, int max_pages, int max_context) { return max_context / c->page_size < max_pages ? max_context / c->page_size : max_pages; }

bool sparse_ready(const abq_sparse_state &st) { return st.attn.init_success && st.attn.kind == kSparseKind; }

} // namespace

} // namespace abq

using namespace abq;

extern "C" {

abq_status abq_rotary_apply(const abq_rotary *rotary, const abq_rows *q, const abq_rows *q_out, int heads, const abq_rows *k, const abq_rows *k_out,
                            int kv_heads, int head_dim, int dtype, const int32_t *positions, int64_t position_stride, void *stream)
{
    if (!q || q->rows < 0 || !dtype_valid(dtype) || head_dim <= 0)
        return ABQ_ERR_INVALID_ARG;
    if (head_dim % 16 || head_dim > 256)
        return ABQ_ERR_UNSUPPORTED;
    abq_status s;
    if ((s = check_rotary(rotary, head_dim, positions, position_stride, q->rows)) != ABQ_OK ||
        (s = check_turned(q, q_out, q->rows, heads, head_dim)) != ABQ_OK || (k && (s = check_turned(k, k_out, q->rows, kv_heads, head_dim)) != ABQ_OK))
        return s;
    if (k && crossed(q, q_out, k, k_out))
        return ABQ_ERR_INVALID_ARG;
    RotaryCall c = {};
    c.rotary = *rotary;
    c.q = *q;
    c.q_out = *q_out;
    c.heads[0] = heads;
    if (k) {
        c.k = *k;
        c.k_out = *k_out;
        c.heads[1] = kv_heads;
    }
    c.head_dim = head_dim;
    c.dtype = dtype;
    c.tokens = q->rows;
    c.positions = positions;
    c.position_stride = position_stride;
    if ((s = check_turning(c, 0)) != ABQ_OK)
        return s;
    return hip_status(launch_rotary(c, (hipStream_t)stream));
}

abq_status abq_kv_append_rotary(const abq_kv_cache *cache, const abq_rotary *rotary, const abq_rows *q, const abq_rows *q_out, int heads,
                                const abq_rows *k, const abq_rows *k_out, const abq_rows *v, int dtype, const int32_t *positions,
                                int64_t position_stride, const int32_t *slots, void *stream)
{
    abq_status s = check_cache(cache);
    if (s != ABQ_OK)
        return s;
    if (!k || !v || k->rows < 0 || !dtype_valid(dtype) || (k->rows && !slots) || !q != !q_out)
        return ABQ_ERR_INVALID_ARG;
    if ((s = check_rotary(rotary, cache->head_dim, positions, position_stride, k->rows)) != ABQ_OK ||
        (s = check_rows(v, k->rows, cache->kv_heads, cache->head_dim)) != ABQ_OK ||
        (s = k_out ? check_turned(k, k_out, k->rows, cache->kv_heads, cache->head_dim) : check_rows(k, k->rows, cache->kv_heads, cache->head_dim)) != ABQ_OK ||
        (q && (s = check_turned(q, q_out, k->rows, heads, cache->head_dim)) != ABQ_OK))
        return s;
    if (begins_on(k_out, v) || begins_on(q_out, v) || crossed(q, q_out, k, k_out))
        return ABQ_ERR_INVALID_ARG;
    RotaryCall c = {};
    c.rotary = *rotary;
    if (q) {
        c.q = *q;
        c.q_out = *q_out;
        c.heads[0] = heads;
    }
    c.k = *k;
    if (k_out)
        c.k_out = *k_out;
    c.heads[1] = cache->kv_heads;
    c.v = *v;
    c.head_dim = cache->head_dim;
    c.dtype = dtype;
    c.tokens = k->rows;
    c.positions = positions;
    c.position_stride = position_stride;
    c.cache = cache;
    c.slots = slots;
    if (k->rows > 0x7ffffff0)
        return ABQ_ERR_TOO_LARGE;
    if ((s = check_turning(c, product((k->rows + 3) / 4 * 2, cache->kv_heads, 1) / 4 + 1)) != ABQ_OK)
        return s;
    return hip_status(launch_rotary(c, (hipStream_t)stream));
}

abq_status abq_kv_pages_fork(const abq_kv_pages *pages, const int32_t *parents, void *stream)
{
    const abq_status s = check_pages(pages);
    if (s != ABQ_OK)
        return s;
    if (!parents)
        return ABQ_ERR_INVALID_ARG;
    return hip_status(launch_pages_fork(*pages, parents, (hipStream_t)stream));
}

abq_status abq_kv_pages_extend(const abq_kv_pages *pages, const int32_t *counts, int32_t *slots, int64_t rows, int32_t *starts, int32_t *granted,
                               int32_t *copies, void *stream)
{
    const abq_status s = check_pages(pages);
    if (s != ABQ_OK)
        return s;
    if (!counts || rows < 0 || (rows && !slots) || !starts || !granted || !copies)
        return ABQ_ERR_INVALID_ARG;
    if (rows > 0x7ffffff0)
        return ABQ_ERR_TOO_LARGE;
    return hip_status(launch_pages_extend(*pages, counts, slots, rows, starts, granted, copies, (hipStream_t)stream));
}

abq_status abq_kv_pages_compact(const abq_kv_pages *pages, int32_t *moves, void *stream)
{
    const abq_status s = check_pages(pages);
    if (s != ABQ_OK)
        return s;
    if (!moves && pages->num_pages > 1)
        return ABQ_ERR_INVALID_ARG;
    if (product(pages->seqs, pages->max_pages, 1) > kMostBlocks * 256 - 256)
        return ABQ_ERR_TOO_LARGE;
    return hip_status(launch_pages_compact(*pages, moves, (hipStream_t)stream));
}

abq_status abq_kv_copy_pages(const abq_kv_cache *cache, const abq_kv_bounds *bounds, const int32_t *pairs, int64_t count, void *stream)
{
    abq_status s = check_cache(cache);
    if (s != ABQ_OK)
        return s;
    if (count < 0 || (count && !pairs))
        return ABQ_ERR_INVALID_ARG;
    if (bounds && (s = check_bounds(bounds)) != ABQ_OK)
        return s;
    if (count > kMostBlocks)
        return ABQ_ERR_TOO_LARGE;
    return hip_status(launch_copy_pages(*cache, bounds, pairs, count, (hipStream_t)stream));
}

size_t abq_kv_bound_codes_bytes(const abq_kv_cache *c)
{
    return cache_sizes_valid(c) ? (size_t)c->num_pages * c->kv_heads * 2 * c->head_dim : 0;
}

size_t abq_kv_bound_scales_bytes(const abq_kv_cache *c) { return cache_sizes_valid(c) ? (size_t)c->num_pages * c->kv_heads * sizeof(float) : 0; }

abq_status abq_kv_bound(const abq_kv_cache *cache, const abq_kv_bounds *bounds, const int32_t *slots, int64_t count, void *stream)
{
    abq_status s = check_cache(cache);
    if (s != ABQ_OK || (s = check_bounds(bounds)) != ABQ_OK)
        return s;
    if (count < 0 || (count && !slots))
        return ABQ_ERR_INVALID_ARG;
    // (workgroups in eights)
    if (product((count - 1) / bound_slots(*cache, count) + 1, (cache->kv_heads + 3) / 4, 1) > kMostBlocks / 8 * 8)
        return ABQ_ERR_TOO_LARGE;
    return hip_status(launch_kv_bound(*cache, *bounds, slots, count, (hipStream_t)stream));
}

size_t abq_attn_choose_workspace_bytes(const abq_kv_cache *cache, int max_pages, int seqs, int max_q, int max_context)
{
    if (!cache_sizes_valid(cache) || max_pages <= 0 || max_pages > kMostChosen || seqs <= 0 || max_q <= 0 || max_context < 0)
        return 0;
    return choose_workspace_bytes(seqs, max_q, cache->kv_heads, max_pages, likely_pages(cache, max_pages, max_context));
}

abq_status abq_attn_choose(const abq_kv_cache *cache, const abq_kv_bounds *bounds, const abq_rows *q, int dtype, int heads, const int32_t *page_table,
                           int max_pages, const int32_t *context, const int32_t *q_starts, int seqs, int max_q, int max_context, int first, int last, int count,
                           int32_t *blocks, void *workspace, size_t workspace_bytes, void *stream)
{
    abq_status s = check_cache(cache);
    if (s != ABQ_OK || (s = check_bounds(bounds)) != ABQ_OK)
        return s;
    if (!q || q->rows < 0 || !dtype_valid(dtype) || heads <= 0 || heads % cache->kv_heads || !page_table || max_pages <= 0 || !context || !q_starts ||
        seqs <= 0 || max_q <= 0 || max_context < 0 || first < 0 || last < 0 || count <= 0 || (int64_t)first + last > count || (q->rows && !blocks) ||
        (workspace_bytes && !workspace) || !aligned(workspace, 4))
        return ABQ_ERR_INVALID_ARG;
    if ((s = check_rows(q, q->rows, heads, cache->head_dim)) != ABQ_OK)
        return s;
    if (max_pages > kMostChosen || count > kMostChosen || q->rows > 0x7ffffff0 || (int64_t)max_pages * cache->page_size > 0x7fffffff - 64 ||
        product(product(seqs, max_q, cache->kv_heads), 1024, 1) > kMostThreads)
        return ABQ_ERR_TOO_LARGE;
    return hip_status(launch_attn_choose({*cache, *bounds, *q, dtype, heads, page_table, context, q_starts, max_pages, seqs, max_q, first, last, count,
                                          likely_pages(cache, max_pages, max_context), blocks, workspace, workspace_bytes},
                                         (hipStream_t)stream));
}

abq_status abq_attn_sparse_init(const abq_kv_cache *cache, const abq_rows *q, const abq_rows *out, int dtype, int heads, const int32_t *page_table,
                                int max_pages, const int32_t *context, const int32_t *q_starts, const uint64_t *mask, const int32_t *blocks, int count,
                                int seqs, int max_q, int max_context, float scale, abq_sparse_state *state)
{
    if (!state)
        return ABQ_ERR_INVALID_ARG;
    memset(state, 0, sizeof *state);
    abq_sparse_state st = {};
    abq_status s = abq_attn_tree_init(cache, q, out, dtype, heads, page_table, max_pages, context, q_starts, mask, seqs, max_q, max_context, scale, &st.attn);
    if (s != ABQ_OK)
        return s;
    if ((q->rows && !blocks) || count <= 0)
        return ABQ_ERR_INVALID_ARG;
    if (count > kMostChosen || product(product(seqs, max_q, cache->kv_heads) + 8, (heads / cache->kv_heads + 15) / 16, 1) > kMostThreads / 512)
        return ABQ_ERR_TOO_LARGE;
    st.attn.kind = kSparseKind;
    st.blocks = blocks;
    st.count = count;
    plan_attn_sparse(&st, 1);
    *state = st;
    return ABQ_OK;
}

size_t abq_attn_sparse_workspace_bytes(const abq_sparse_state *state)
{
    if (!state || !sparse_ready(*state))
        return 0;
    abq_sparse_state best = *state;
    plan_attn_sparse(&best, kMostParts);
    return attn_parts_bytes(best.attn, best.attn.parts);
}

abq_status abq_attn_sparse_set_workspace(abq_sparse_state *state, void *workspace, size_t bytes)
{
    if (!state)
        return ABQ_ERR_INVALID_ARG;
    if (!sparse_ready(*state))
        return ABQ_ERR_NOT_INITIALIZED;
    if ((bytes && !workspace) || !aligned16(workspace))
        return ABQ_ERR_INVALID_ARG;
    const size_t one = attn_parts_bytes(state->attn, 2) / 2;
    size_t parts = workspace && one ? bytes / one : 1;
    parts = parts < 2 ? 1 : parts > kMostParts ? kMostParts : parts;
    state->attn.workspace = workspace;
    state->attn.workspace_bytes = bytes;
    plan_attn_sparse(state, (int)parts);
    return ABQ_OK;
}

abq_status abq_attn_sparse_exec(const abq_sparse_state *state, void *stream)
{
    if (!state)
        return ABQ_ERR_INVALID_ARG;
    if (!sparse_ready(*state))
        return ABQ_ERR_NOT_INITIALIZED;
    return state->attn.q.rows == 0 ? ABQ_OK : hip_status(launch_attn_sparse(*state, (hipStream_t)stream));
}

} // extern "C"
