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
 * Rotary positions
 *
 * Of every head's first rotary_dim elements, pair i (of rotary_dim / 2) is turned by its token's position:
 *   t = positions[axis[i]][token] * turns[i],  c = cos(2 pi t),  s = sin(2 pi t),  (a, b) -> (a c - b s, b c + a s)
 * The pair's elements are i and i + rotary_dim / 2, or 2 i and 2 i + 1 if interleaved.  t is a product in fp64, cosine, sine and
 * the turned elements are fp64 and are rounded to fp32 and then to the type: a row comes out the same wherever it stands, and
 * positions of any size keep their angle to 2^-52 of the position's number of turns.  The other elements are copied.
 * ------------------------------------------------------------------------------------- */
typedef struct abq_rotary {
    int rotary_dim;      /* a multiple of 16, at most head_dim */
    int axes;            /* 1 .. 8: rows of positions, such as time, height and width */
    int interleaved;
    const double *turns; /* device, [rotary_dim / 2]: revolutions per position, base^(-2 i / rotary_dim) / (2 pi) and whatever scaling a model has */
    const int32_t *axis; /* device, [rotary_dim / 2], each 0 .. axes - 1 (others count as the nearest of these); NULL: all 0 */
} abq_rotary;

/* Turns rows of q into q_out and of k into k_out: into the same rows, in place, or others; but for that nothing that is written may
 * overlap anything else that is read or written (results that begin where other rows do are refused).  k (and k_out) may be NULL.  positions: device int32, axis a of token i at
 * positions[a * position_stride + i]; position_stride >= the number of rows where there are several axes.  head_dim: a multiple of 16, at most 256. */
abq_status abq_rotary_apply(const abq_rotary *rotary, const abq_rows *q, const abq_rows *q_out, int heads, const abq_rows *k, const abq_rows *k_out,
                            int kv_heads, int head_dim, int dtype, const int32_t *positions, int64_t position_stride, void *stream);

/* abq_rotary_apply and abq_kv_append in one launch: q is turned into q_out (both may be NULL), k into k_out if that is not NULL, and the
 * turned rows of k, as they are rounded to dtype, and those of v are quantised into the cache as abq_kv_append does.  v must not overlap
 * q_out or k_out. */
abq_status abq_kv_append_rotary(const abq_kv_cache *cache, const abq_rotary *rotary, const abq_rows *q, const abq_rows *q_out, int heads,
                                const abq_rows *k, const abq_rows *k_out, const abq_rows *v, int dtype, const int32_t *positions,
                                int64_t position_stride, const int32_t *slots, void *stream);

/* ---------------------------------------------------------------------------------------
 * Pages of sequences
 *
 * Which pages of the cache hold which sequence's tokens, kept on the device, so that steps of beam search, of drafts or of ordinary
 * decoding can be captured whole.  One such table serves the caches of all layers, which have num_pages pages of page_size tokens each.
 * Between calls: table[s * max_pages + j] is the page of tokens j * page_size .. of sequence s for j below
 * ceil(lengths[s] / page_size), and -1 behind; refs[p] is the number of entries that name page p, 0 for a free one.  Initially every
 * entry is -1, lengths and refs are 0.  Sequences may share pages.  The calls keep to the arrays whatever these hold.
 * ------------------------------------------------------------------------------------- */
typedef struct abq_kv_pages {
    int seqs;      /* at most 8192 */
    int max_pages; /* of a sequence; at most 2^22 - 3, and max_pages * page_size < 2^31 - 64 */
    int page_size; /* as in abq_kv_cache */
    int num_pages;
    int32_t *table, *lengths, *refs; /* device: [seqs][max_pages], [seqs], [num_pages] */
} abq_kv_pages;

/* Sequence s becomes what sequence parents[s] was before the call (device, [seqs]): it has its length and shares its pages.  A parent
 * outside 0 .. seqs - 1, such as -1, leaves the sequence empty.  Pages that nobody names any more are free. */
abq_status abq_kv_pages_fork(const abq_kv_pages *pages, const int32_t *parents, void *stream);

/* Gives sequence s room for counts[s] more tokens (device, [seqs]), or takes -counts[s] of its last tokens away.  Tokens to be written in a
 * page that other entries name as well go to a copy of it.  Pages that were free before the call are handed out lowest first, in the order of the
 * sequences, a copy's page before the further ones.  A sequence that would need more than max_pages is left as it is; so are the first
 * one for which the free pages do not suffice and those behind it that need any.  The search for free pages begins at the first page: a call
 * that needs any takes the longer the more occupied ones lie in front of them.  Device arrays, written whole:
 *   starts  [seqs + 1]  where the sequences' new tokens begin, one behind the other: sums of the positive counts (as q_starts), at most 2^31 - 1
 *   granted [seqs]      counts[s], 0 for a sequence that was left as it was, -(tokens taken away)
 *   copies  [seqs][2]   pages (from, to) to be copied in every layer's cache before anything is written to it, or -1, -1
 *   slots   [rows]      the new tokens' places, for abq_kv_append; -1 for tokens that were not granted and behind the last one */
abq_status abq_kv_pages_extend(const abq_kv_pages *pages, const int32_t *counts, int32_t *slots, int64_t rows, int32_t *starts, int32_t *granted,
                               int32_t *copies, void *stream);

/* Moves pages so that the live ones are the first: of n live pages, those behind page n - 1, in order, take the places of the free ones before it,
 * in order.  moves (device, [num_pages / 2][2]): pages (from, to) to be copied in every layer's cache, -1, -1 behind the last. */
abq_status abq_kv_pages_compact(const abq_kv_pages *pages, int32_t *moves, void *stream);

/* Bounds of the keys of every page: see abq_kv_bound */
typedef struct abq_kv_bounds {
    int8_t *codes; /* [page][head][2][head_dim]: of the largest, of the smallest; abq_kv_bound_codes_bytes, 16-byte aligned */
    float *scales; /* [page][head]; abq_kv_bound_scales_bytes */
} abq_kv_bounds;

/* Copies page pairs[i][0] to page pairs[i][1], i = 0 .. count - 1 (device; -1, or anything outside the cache: nothing is copied), with its bounds
 * if there are any (bounds may be NULL).  No page may be written twice in one call, or written and read, unless it is copied to itself. */
abq_status abq_kv_copy_pages(const abq_kv_cache *cache, const abq_kv_bounds *bounds, const int32_t *pairs, int64_t count, void *stream);

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

/* ---------------------------------------------------------------------------------------
 * Attention to chosen pages
 *
 * Every query looks at a few pages of its context, chosen by a bound of the scores that it can have there, and at the newest
 * tokens.  The bound of a page and key head holds the largest and the smallest of each channel of its keys, as the cache
 * holds them in fp32, 2 head_dim numbers that are quantised as one symmetric row of 8 bits: signed codes hi, lo, and a scale.
 * ------------------------------------------------------------------------------------- */
size_t abq_kv_bound_codes_bytes(const abq_kv_cache *cache);
size_t abq_kv_bound_scales_bytes(const abq_kv_cache *cache);

/* Writes the bounds of the pages whose last slot is among slots[0 .. count - 1] (device; slots outside the cache are passed over): called
 * with the slots of each abq_kv_append behind it, it leaves bounds of all pages that are complete. */
abq_status abq_kv_bound(const abq_kv_cache *cache, const abq_kv_bounds *bounds, const int32_t *slots, int64_t count, void *stream);

/* Chooses pages.  Sequence s has context[s] tokens in the cache and rows q_starts[s] .. q_starts[s + 1] - 1 of q, of which the first max_q
 * are dealt with.  Of its n = context[s] / page_size complete pages (at most max_pages), each row and key head gets `count`: all if there are
 * no more, else the first `first`, the last `last` and those with the largest scores, lower pages before higher ones where scores are equal;
 * first + last <= count.  With q quantised per row and head as a symmetric row of 8 bits, codes c and scale d,
 *   score = max over the heads of the group (fp32(sum max(c, 0) hi + min(c, 0) lo) * d) * (the bound's scale),   in fp32,
 * at least the largest q . k of the page but for the roundings to 8 bits.  A page that is not in the cache has the lowest score.
 * blocks (device, int32 [rows of q][kv_heads][count]): the pages' numbers in the sequence, ascending, -1 behind the last.  Rows that are not
 * dealt with keep what they hold.  max_pages <= 32768; max_context only guides how the work is split.  workspace: NULL, or a device buffer,
 * 4-byte aligned, of abq_attn_choose_workspace_bytes (0: none is used), which nothing else may use while the call is under way; a smaller one is
 * as none.  The choice is the same with and without. */
size_t abq_attn_choose_workspace_bytes(const abq_kv_cache *cache, int max_pages, int seqs, int max_q, int max_context);
abq_status abq_attn_choose(const abq_kv_cache *cache, const abq_kv_bounds *bounds, const abq_rows *q, int dtype, int heads, const int32_t *page_table,
                           int max_pages, const int32_t *context, const int32_t *q_starts, int seqs, int max_q, int max_context, int first, int last, int count,
                           int32_t *blocks, void *workspace, size_t workspace_bytes, void *stream);

/* Attention of drafted tokens as in abq_attn_tree_init, but of the context, row i and key head h see only the tokens of pages
 * blocks[i][h][0 .. count - 1] (numbers that are not those of complete pages of the context name none; a page that is named
 * twice counts twice) and those behind the last complete page.  count <= 32768, and best not much more than there are pages to name. */
typedef struct abq_sparse_state {
    abq_attn_state attn;
    const int32_t *blocks;
    int count;
} abq_sparse_state;
abq_status abq_attn_sparse_init(const abq_kv_cache *cache, const abq_rows *q, const abq_rows *out, int dtype, int heads, const int32_t *page_table,
                                int max_pages, const int32_t *context, const int32_t *q_starts, const uint64_t *mask, const int32_t *blocks, int count,
                                int seqs, int max_q, int max_context, float scale, abq_sparse_state *state);

/* As abq_attn_workspace_bytes, abq_attn_set_workspace and abq_attn_exec */
size_t abq_attn_sparse_workspace_bytes(const abq_sparse_state *state);
abq_status abq_attn_sparse_set_workspace(abq_sparse_state *state, void *workspace, size_t bytes);
abq_status abq_attn_sparse_exec(const abq_sparse_state *state, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ABQ_ATTENTION_H */
