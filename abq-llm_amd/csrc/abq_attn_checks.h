// Checks of arguments that the host API of attention (abq_attention.hip) and that of what a decoding step needs around it
// (abq_decoding.hip) share.
#pragma once
#include <stdint.h>

#include "abq_attn.h"

namespace abq {

// a * b * c, none of them negative, or more than any limit here where that does not fit
inline int64_t product(int64_t a, int64_t b, int64_t c)
{
    int64_t x;
    return __builtin_mul_overflow(a, b, &x) || __builtin_mul_overflow(x, c, &x) ? INT64_MAX : x;
}

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// written: rows of a result, which may not lie on one another
inline abq_status check_rows(const abq_rows *r, int64_t rows, int heads, int head_dim, bool written = false)
{
    if (!r || r->rows != rows || (rows && !r->data) || !aligned16(r->data) || r->row_stride % 8 || r->head_stride % 8)
        return ABQ_ERR_INVALID_ARG;
    if (r->row_stride < 0 || r->head_stride < 0 || (heads > 1 && r->head_stride < head_dim) || (written && rows > 1 && r->row_stride < head_dim))
        return ABQ_ERR_INVALID_ARG;
    return ABQ_OK;
}

inline bool cache_sizes_valid(const abq_kv_cache *c)
{
    return c && (c->bits == 8 || c->bits == 4) && (c->head_dim == 64 || c->head_dim == 128) && c->kv_heads > 0 && c->num_pages > 0 &&
           c->page_size >= 16 && c->page_size <= 4096 && (c->page_size & (c->page_size - 1)) == 0 &&
           (int64_t)c->num_pages * c->page_size <= 0x7fffffff && c->kv_heads <= 65536;
}

inline abq_status check_cache(const abq_kv_cache *c)
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

} // namespace abq
