/*
 * abq_attention.h -- C ABI of attention on a quantised key / value cache, the part of a decoder layer that stands between
 * the QKV and the output GEMM of abq_gemm.h.  Same library, same conventions: plain pointers and sizes, device pointers
 * valid on the current HIP device, `stream` a hipStream_t passed as void*, status codes of abq_gemm.h, no device memory
 * allocated, no global state.  Everything is stream ordered; index arrays (slots, page tables, lengths, masks) are read by
 * the kernels, so a captured HIP graph replays with whatever they hold then.
 *
 * The reference engine leaves attention to FasterTransformer's layers (layers/attention_layers/GptContextAttentionLayer.cc,
 * DecoderSelfAttentionLayer.cc) on a cache of the activations' type.  Keys and values are quantised per token and head with
 * the quantiser of its calibration (algorithm/quantize/quantizer.py:111-179), as abq_quant_pack_f16 does with activations.
 */
#ifndef ABQ_ATTENTION_H
#define ABQ_ATTENTION_H

#include "abq_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum abq_dtype {
    ABQ_F16 = 0,
    ABQ_BF16 = 1
} abq_dtype;

/* A device matrix of rows (tokens) of heads: element d of head h of row r stands at data[r * row_stride + h * head_stride
 * + d], strides in elements.  Rows of heads are read and written 16 bytes at a time: data must be 16-byte aligned and both
 * strides multiples of 8 (a slice of a fused QKV result is one), head_stride at least head_dim where there are several heads, and
 * in results row_stride as well where there are several rows (rows that are read may repeat).  Nothing outside rows
 * 0 .. rows - 1 is touched. */
typedef struct abq_rows {
    void *data;
    int64_t rows;
    int64_t row_stride, head_stride;
} abq_rows;

/* ---------------------------------------------------------------------------------------
 * Quantised cache
 *
 * Pages of page_size tokens (a power of two, 16 .. 4096), each holding all kv_heads.  A token's place is its slot,
 * page * page_size + offset in the page; num_pages * page_size must stay below 2^31.  A row x[0 .. head_dim) of a token and
 * head becomes unsigned codes u and a scale (and a zero point), the row's value then being scale * (u - zero):
 *   symmetric:  scale = clamp(absmax / (2^(bits-1) - 1), 1e-5, 1e4), zero = 2^(bits-1),
 *               u = clamp(rint(x / scale), -2^(bits-1), 2^(bits-1) - 1) + zero
 *   otherwise:  scale = clamp((max - min) / (2^bits - 1), 1e-5, 1e4), zero = rint(clamp(-min / scale, -1e4, 1e4)),
 *               u = clamp(rint(x / scale) + zero, 0, 2^bits - 1)
 * in fp32, half to even, quotients correctly rounded.  Infinite elements get the outermost code, NaN elements any; scales
 * are finite whatever the row holds.
 *
 * Layout, R = head_dim * bits / 8 bytes per row, token t of a page:
 *   k_codes  [page][head][t][R]               8 bits: byte d.  4 bits: the eight codes of d = 8 w .. 8 w + 7 in word w, in
 *                                             nibbles 0, 4, 1, 5, 2, 6, 3, 7
 *   v_codes  [page][head][t / 4][R][4]        four tokens beside each other: byte column c of token t at [t / 4][c][p(t % 4)].
 *                                             8 bits: c = d, p = 0, 1, 2, 3.  4 bits: low nibble d = c, high nibble
 *                                             d = c + head_dim / 2, p = 0, 2, 1, 3
 *   k_scales, v_scales  symmetric [page][head][page_size], otherwise [page][head][2][page_size]: scales, then zero points
 * ------------------------------------------------------------------------------------- */
typedef struct abq_kv_cache {
    int bits;      /* 8 or 4 */
    int symmetric; /* 0: rows have zero points */
    int kv_heads;
    int head_dim;  /* 64 or 128 */
    int page_size;
    int num_pages;
    void *k_codes, *v_codes;     /* abq_kv_codes_bytes each, 16-byte aligned */
    float *k_scales, *v_scales;  /* abq_kv_scales_bytes each, 16-byte aligned */
} abq_kv_cache;

/* Bytes of one of the two code arrays (scale arrays); 0 if the sizes are not valid.  The pointers are not looked at. */
size_t abq_kv_codes_bytes(const abq_kv_cache *cache);
size_t abq_kv_scales_bytes(const abq_kv_cache *cache);

/* Quantises row i of k and v and writes it at slots[i], i = 0 .. k->rows - 1 (= v->rows).  A slot that is negative or beyond
 * the cache drops its row.  Slots of one call must differ from each other (of two rows for one slot, parts of either may
 * stay); other slots keep what they hold.  rows may be 0. */
abq_status abq_kv_append(const abq_kv_cache *cache, const abq_rows *k, const abq_rows *v, int dtype, const int32_t *slots, void *stream);

/* The inverse: row i of k and v receives the values that slots[i] holds, scale * (u - zero) in fp32 rounded once to dtype;
 * zeros for a slot outside the cache. */
abq_status abq_kv_read(const abq_kv_cache *cache, const abq_rows *k, const abq_rows *v, int dtype, const int32_t *slots, void *stream);

/* ---------------------------------------------------------------------------------------
 * Attention
 *
 * out[i][h] = sum_t p[t] v[t][h / group] over the tokens t that query i sees, p = softmax(scale * q[i][h] . k[t][h / group]),
 * group = heads / kv_heads.  Scores, statistics and sums are fp32; a query that sees nothing gets zeros; what a query does
 * not see never reaches its result, infinities and NaN included.  A finite result beyond dtype's largest becomes that one.
 *
 * As with a GEMM, a caller-owned state is filled once (init) and run any number of times (exec).
 * ------------------------------------------------------------------------------------- */
typedef struct abq_attn_state {
    int init_success;
    int kind;  /* 1: whole prompts, 2: drafts on a cache */
    int dtype; /* abq_dtype of q, out and, for prompts, k and v */
    int heads, kv_heads, head_dim;
    int seqs, max_q, max_k;
    float scale;
    abq_rows q, k, v, out;
    const int32_t *q_starts, *k_starts;
    /* drafts on a cache */
    abq_kv_cache cache;
    const int32_t *page_table, *context;
    const uint64_t *mask;
    int max_pages;
    /* how it runs: parts that a sequence's tokens are split into, query rows of a workgroup */
    int parts, block_rows;
    void *workspace;
    size_t workspace_bytes;
} abq_attn_state;

/* Causal attention of packed prompts.  Sequence s owns rows q_starts[s] .. q_starts[s + 1] - 1 of q and out and rows
 * k_starts[s] .. k_starts[s + 1] - 1 of k and v (k_starts NULL: the same as q_starts); rows of k and v are at most 2^25
 * elements apart; starts are device arrays of seqs + 1 ascending offsets.  The queries are the last of the sequence's tokens:
 * query i of n sees keys 0 .. m - n + i of m, so with fewer keys than queries the first n - m queries see nothing.  max_q,
 * max_k: bounds of a sequence's queries and keys on the host; queries beyond max_q are not computed and their rows of out stay
 * as they are, max_k only guides how the work is split.  0 < scale <= 2e38.  out must not overlap q, k or v.  A sequence may
 * be empty. */
abq_status abq_attn_prompt_init(const abq_rows *q, const abq_rows *k, const abq_rows *v, const abq_rows *out, int dtype, int heads,
                                int kv_heads, int head_dim, const int32_t *q_starts, const int32_t *k_starts, int seqs, int max_q,
                                int max_k, float scale, abq_attn_state *state);

/* Attention of drafted tokens over the quantised cache.  Sequence s holds context[s] tokens in the cache and behind them its
 * drafts, rows q_starts[s] .. q_starts[s + 1] - 1 of q and out (at most 64), whose keys and values have been appended at the
 * places that follow the context.  Drafts beyond max_q <= 64 are not computed, and their rows of out stay as they are, but
 * they can be seen.  Place t of sequence s is offset t % page_size of page page_table[s * max_pages + t / page_size]; places on
 * pages outside the cache, or beyond max_pages, are not seen.  Draft i sees the context and the drafts j whose bit j is set in
 * mask[q_starts[s] + i] (itself only if its own bit is); mask NULL: drafts 0 .. i, a chain.  One draft per sequence and no
 * mask is ordinary decoding.  max_context only guides how the work is split.  0 < scale <= 2e30. */
abq_status abq_attn_tree_init(const abq_kv_cache *cache, const abq_rows *q, const abq_rows *out, int dtype, int heads,
                              const int32_t *page_table, int max_pages, const int32_t *context, const int32_t *q_starts,
                              const uint64_t *mask, int seqs, int max_q, int max_context, float scale, abq_attn_state *state);

/* Workspace with which the state would run as it runs best: few queries over many tokens are split over the tokens, and the
 * parts' results, held in fp32, are joined by a second launch.  0 if it is not split. */
size_t abq_attn_workspace_bytes(const abq_attn_state *state);

/* Hands a caller-owned device buffer, 16-byte aligned, to the state.  Without one, or with a smaller one than
 * abq_attn_workspace_bytes, the tokens are split into fewer parts, or not.  Results may differ in the last bits with the number
 * of parts.  While a call is under way nothing else may use the buffer. */
abq_status abq_attn_set_workspace(abq_attn_state *state, void *workspace, size_t bytes);

abq_status abq_attn_exec(const abq_attn_state *state, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ABQ_ATTENTION_H */
