// Host side of the C ABI declared in include/abq_attention.h: argument checks, sizes, and the choice of how the work is laid
// out.  No entry point allocates device or host memory.
#include "abq_attention.h"

#include <hip/hip_runtime.h>
#include <math.h>
#include <string.h>

#include "abq_attn.h"

namespace abq {

namespace {

constexpr int kPromptKind = 1, kTreeKind = 2;

// A tile of keys or values is addressed from its first row in 32 bits: 63 strides of 2-byte elements and a row
constexpr int64_t kMostTileStride = 1 << 25;

// Scales that fp32 holds times log2(e), and for drafts times a token's scale and zero point, of up to 1e4 each, as well
constexpr float kMostPromptScale = 2e38f, kMostTreeScale = 2e30f;

// a * b * c, none of them negative, or more than any limit here where that does not fit
int64_t product(int64_t a, int64_t b, int64_t c)
{
    int64_t x;
    return __builtin_mul_overflow(a, b, &x) || __builtin_mul_overflow(x, c, &x) ? INT64_MAX : x;
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// written: rows of a result, which may not lie on one another
abq_status check_rows(const abq_rows *r, int64_t rows, int heads, int head_dim, bool written = false)
{
    if (!r || r->rows != rows || (rows && !r->data) || !aligned16(r->data) || r->row_stride % 8 || r->head_stride % 8)
        return ABQ_ERR_INVALID_ARG;
    if (r->row_stride < 0 || r->head_stride < 0 || (heads > 1 && r->head_stride < head_dim) || (written && rows > 1 && r->row_stride < head_dim))
        return ABQ_ERR_INVALID_ARG;
    return ABQ_OK;
}

bool cache_sizes_valid(const abq_kv_cache *c)
{
    return c && (c->bits == 8 || c->bits == 4) && (c->head_dim == 64 || c->head_dim == 128) && c->kv_heads > 0 && c->num_pages > 0 &&
           c->page_size >= 16 && c->page_size <= 4096 && (c->page_size & (c->page_size - 1)) == 0 &&
           (int64_t)c->num_pages * c->page_size <= 0x7fffffff && c->kv_heads <= 65536;
}

abq_status check_cache(const abq_kv_cache *c)
{
    if (!c)
        return ABQ_ERR_INVALID_ARG;
    if ((c->bits != 8 && c->bits != 4) || (c->head_dim != 64 && c->head_dim != 128))
        return ABQ_ERR_UNSUPPORTED;
    if (!cache_sizes_valid(c) || !c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales || !aligned16(c->k_codes) ||
        !aligned16(c->v_codes) || !aligned16(c->k_scales) || !aligned16(c->v_scales))
        return ABQ_ERR_INVALID_ARG;
    return ABQ_OK;
}

abq_status check_cache_call(const abq_kv_cache *c, const abq_rows *k, const abq_rows *v, int dtype, const int32_t *slots, bool written)
{
    abq_status s = check_cache(c);
    if (s != ABQ_OK)
        return s;
    if (!k || !v || (dtype != ABQ_F16 && dtype != ABQ_BF16) || k->rows < 0 || (k->rows && !slots))
        return ABQ_ERR_INVALID_ARG;
    if ((s = check_rows(k, k->rows, c->kv_heads, c->head_dim, written)) != ABQ_OK ||
        (s = check_rows(v, k->rows, c->kv_heads, c->head_dim, written)) != ABQ_OK)
        return s;
    if (k->rows > 0x7ffffff0 || (k->rows + 3) / 4 * 2 * c->kv_heads > 4 * kMostBlocks - 4)
        return ABQ_ERR_TOO_LARGE;
    return ABQ_OK;
}

// The part of an initialisation that both kinds share; on success the state holds everything but what tells them apart
abq_status init_common(int kind, const abq_rows *q, const abq_rows *out, int dtype, int heads, int kv_heads, int head_dim, const int32_t *q_starts,
                       int seqs, int max_q, float scale, abq_attn_state *st)
{
    if (!q || !out || !q_starts || (dtype != ABQ_F16 && dtype != ABQ_BF16) || heads <= 0 || kv_heads <= 0 || seqs <= 0 || max_q <= 0 ||
        q->rows < 0 || !(scale > 0) || !(scale <= (kind == kTreeKind ? kMostTreeScale : kMostPromptScale)))
        return ABQ_ERR_INVALID_ARG;
    if (head_dim != 64 && head_dim != 128)
        return ABQ_ERR_UNSUPPORTED;
    if (heads % kv_heads)
        return ABQ_ERR_INVALID_ARG;
    abq_status s;
    if ((s = check_rows(q, q->rows, heads, head_dim)) != ABQ_OK || (s = check_rows(out, q->rows, heads, head_dim, true)) != ABQ_OK)
        return s;
    if (q->rows > 0x7ffffff0 || product(q->rows, heads, 1) > 1ll << 42) // (so that bytes of a workspace fit 64 bits)
        return ABQ_ERR_TOO_LARGE;
    st->kind = kind;
    st->dtype = dtype;
    st->heads = heads;
    st->kv_heads = kv_heads;
    st->head_dim = head_dim;
    st->seqs = seqs;
    st->max_q = max_q;
    st->scale = scale;
    st->q = *q;
    st->out = *out;
    st->q_starts = q_starts;
    return ABQ_OK;
}

void plan(abq_attn_state *st, int most_parts)
{
    if (st->kind == kTreeKind)
        plan_attn_tree(st, most_parts);
    else
        plan_attn_prompt(st, most_parts);
}

constexpr int kMostParts = 4096;

} // namespace

} // namespace abq

using namespace abq;

extern "C" {

size_t abq_kv_codes_bytes(const abq_kv_cache *c)
{
    return cache_sizes_valid(c) ? (size_t)c->num_pages * c->page_size * c->kv_heads * c->head_dim * c->bits / 8 : 0;
}

size_t abq_kv_scales_bytes(const abq_kv_cache *c)
{
    return cache_sizes_valid(c) ? (size_t)c->num_pages * c->page_size * c->kv_heads * (c->symmetric ? 1 : 2) * sizeof(float) : 0;
}

abq_status abq_kv_append(const abq_kv_cache *c, const abq_rows *k, const abq_rows *v, int dtype, const int32_t *slots, void *stream)
{
    const abq_status s = check_cache_call(c, k, v, dtype, slots, false);
    return s != ABQ_OK ? s : hip_status(launch_kv_append(*c, *k, *v, dtype, slots, (hipStream_t)stream));
}

abq_status abq_kv_read(const abq_kv_cache *c, const abq_rows *k, const abq_rows *v, int dtype, const int32_t *slots, void *stream)
{
    const abq_status s = check_cache_call(c, k, v, dtype, slots, true);
    return s != ABQ_OK ? s : hip_status(launch_kv_read(*c, *k, *v, dtype, slots, (hipStream_t)stream));
}

abq_status abq_attn_prompt_init(const abq_rows *q, const abq_rows *k, const abq_rows *v, const abq_rows *out, int dtype, int heads, int kv_heads,
                                int head_dim, const int32_t *q_starts, const int32_t *k_starts, int seqs, int max_q, int max_k, float scale,
                                abq_attn_state *state)
{
    if (!state)
        return ABQ_ERR_INVALID_ARG;
    memset(state, 0, sizeof *state);
    abq_status s = init_common(kPromptKind, q, out, dtype, heads, kv_heads, head_dim, q_starts, seqs, max_q, scale, state);
    if (s != ABQ_OK)
        return s;
    if (!k || !v || max_k <= 0 || k->rows < 0)
        return ABQ_ERR_INVALID_ARG;
    if ((s = check_rows(k, k->rows, kv_heads, head_dim)) != ABQ_OK || (s = check_rows(v, k->rows, kv_heads, head_dim)) != ABQ_OK)
        return s;
    if (!k_starts && k->rows != q->rows)
        return ABQ_ERR_INVALID_ARG;
    state->k = *k;
    state->v = *v;
    state->k_starts = k_starts ? k_starts : q_starts;
    state->max_k = max_k;
    if (k->rows > 0x7ffffff0 || k->row_stride > kMostTileStride || v->row_stride > kMostTileStride ||
        product(((int64_t)max_q + 31) / 32, heads, seqs) > kMostBlocks)
        return ABQ_ERR_TOO_LARGE;
    plan(state, 1);
    state->init_success = 1;
    return ABQ_OK;
}

abq_status abq_attn_tree_init(const abq_kv_cache *cache, const abq_rows *q, const abq_rows *out, int dtype, int heads, const int32_t *page_table,
                              int max_pages, const int32_t *context, const int32_t *q_starts, const uint64_t *mask, int seqs, int max_q,
                              int max_context, float scale, abq_attn_state *state)
{
    if (!state)
        return ABQ_ERR_INVALID_ARG;
    memset(state, 0, sizeof *state);
    abq_status s = check_cache(cache);
    if (s != ABQ_OK)
        return s;
    s = init_common(kTreeKind, q, out, dtype, heads, cache->kv_heads, cache->head_dim, q_starts, seqs, max_q, scale, state);
    if (s != ABQ_OK)
        return s;
    if (!page_table || !context || max_pages <= 0 || max_context < 0)
        return ABQ_ERR_INVALID_ARG;
    if (max_q > 64 || max_context > 0x7fffffff - 64 || (int64_t)max_pages * cache->page_size > 0x7fffffff - 64)
        return ABQ_ERR_TOO_LARGE;
    state->cache = *cache;
    state->page_table = page_table;
    state->max_pages = max_pages;
    state->context = context;
    state->mask = mask;
    state->max_k = max_context + max_q;
    if (product((int64_t)seqs * cache->kv_heads + 8, ((int64_t)max_q * (heads / cache->kv_heads) + 15) / 16, 1) > kMostBlocks)
        return ABQ_ERR_TOO_LARGE;
    plan(state, 1);
    state->init_success = 1;
    return ABQ_OK;
}

size_t abq_attn_workspace_bytes(const abq_attn_state *state)
{
    if (!state || !state->init_success)
        return 0;
    abq_attn_state best = *state;
    plan(&best, kMostParts);
    return attn_parts_bytes(best, best.parts);
}

abq_status abq_attn_set_workspace(abq_attn_state *state, void *workspace, size_t bytes)
{
    if (!state)
        return ABQ_ERR_INVALID_ARG;
    if (!state->init_success)
        return ABQ_ERR_NOT_INITIALIZED;
    if ((bytes && !workspace) || !aligned16(workspace))
        return ABQ_ERR_INVALID_ARG;
    const size_t one = attn_parts_bytes(*state, 2) / 2;
    size_t parts = workspace && one ? bytes / one : 1;
    parts = parts < 2 ? 1 : parts > kMostParts ? kMostParts : parts;
    state->workspace = workspace;
    state->workspace_bytes = bytes;
    plan(state, (int)parts);
    return ABQ_OK;
}

abq_status abq_attn_exec(const abq_attn_state *state, void *stream)
{
    if (!state)
        return ABQ_ERR_INVALID_ARG;
    if (!state->init_success)
        return ABQ_ERR_NOT_INITIALIZED;
    if (state->q.rows == 0)
        return ABQ_OK;
    return hip_status(state->kind == kTreeKind ? launch_attn_tree(*state, (hipStream_t)stream) : launch_attn_prompt(*state, (hipStream_t)stream));
}

} // extern "C"
