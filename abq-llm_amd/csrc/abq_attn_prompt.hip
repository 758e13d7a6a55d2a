// Causal attention of packed prompts with grouped heads.
//
// A workgroup takes a block of one sequence's queries and one head, a wave 32 queries, and goes over the keys in tiles of 64
// tokens with the running maximum and sum of the softmax.  Both products are taken transposed,
// S^T = K q^T and out^T = V^T P^T (32 x 32 x 16 MFMA): lane (i, h) of the first result holds the scores of query i for tokens
// 8 j + 4 h .. + 3, which are, eight at a time, an operand of the second product as they are, if the values' tokens
// come in the same order; so P never leaves its registers, and a query's statistics are two lanes'.  The values are
// transposed on the way out of LDS (ds_read_b64_tr_b16: four tokens of one element per lane).
//
// Tiles of keys and values are loaded straight into LDS, one tile ahead.  A load places a wave's 64 pieces of 16 bytes one
// behind the other, so the pieces of a row change places by the choice of what each lane loads: keys by the row's number
// (32 rows of one column of pieces lie in different banks), values by the row modulo 4 (so do four rows of four pieces).
//
// P is rounded to the type of the inputs for the second product, which wants both of its operands of one type; its sum is taken
// in fp32 before that (a sum of the rounded weights takes 1 % longer).
//
// Long prompts are bound by the matrix cores, at the clock that the power left to the chip allows: 16384 tokens, 32 heads of 128
// on 8 key heads, bf16, 2.2 TFLOP of what queries see, take 1.97 - 2.11 ms (1.04 - 1.12 PFLOP/s; a large matrix product reaches
// 1.38) with the matrix cores busy in 67 % of clocks, of which there are 1.6 - 1.9 GHz.  Short ones are bound by the chain of
// steps: a tile's 64 tokens take 0.6 us whatever the grid, so 1024 tokens of 32 heads, 16 tiles, 18 - 20 us.
#include "abq_attn.h"
#include "abq_lds_dma.h"

#include <type_traits>

namespace abq {

namespace {

struct PromptArgs {
    abq_rows q, k, v, out;
    const int32_t *q_starts, *k_starts;
    int heads, kv_heads, seqs, max_q, blocks; // blocks: of queries in the longest sequence
    float scale_log2;
    AttnParts parts;
};

constexpr int kTokens = 64; // of a tile

typedef __attribute__((ext_vector_type(4))) short short4v;

template <int DTYPE> __device__ __forceinline__ float16v mfma_32x32x16(uint4 a, uint4 b, float16v c)
{
    if constexpr (DTYPE == ABQ_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8v, a), __builtin_bit_cast(bf16x8v, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8v, a), __builtin_bit_cast(half8v, b), c, 0, 0, 0);
}

// Where piece c of row r of a tile stands in LDS (in pieces of 16 bytes from the row's start)
template <int D> __device__ __forceinline__ int key_piece(int r, int c) { return c ^ (D == 128 ? r & 15 : r >> 1 & 7); }
template <int D> __device__ __forceinline__ int value_piece(int r, int c) { return c ^ (D == 128 ? 4 * (r & 3) : 4 * (r >> 1 & 1)); }

// Of a pair of 16-bit floats, the sign bits of those whose exponent is all ones (adding one to it carries there)
template <int DTYPE> __device__ __forceinline__ uint32_t not_finite(uint32_t pair)
{
    return (DTYPE == ABQ_BF16 ? (pair & 0x7f807f80u) + 0x00800080u : (pair & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}

// KG = 1: the four waves share 128 queries, 32 each.  KG = 2: two waves share 64, and the other two take the other 32 tokens of
// each tile; their results are joined at the end.
template <int DTYPE, int D, int KG> __global__ __launch_bounds__(256, 2) void attn_prompt_kernel(PromptArgs a)
{
    constexpr int kBlock = 128 / KG;            // queries of the workgroup
    constexpr int TT = 2 / KG;                  // a wave's 32-token parts of a tile
    constexpr int kPieces = D / 8;              // of a row
    constexpr int kTile = kTokens * D * 2;      // bytes
    constexpr int kLoads = kTile / 1024 / 4;    // of a wave per tile
    __shared__ __align__(1024) uint8_t lds[4][kTile]; // keys of two tiles, values of two tiles
    __shared__ int odd_values[4];
    static_assert(KG == 1 || 4 * kTile >= 64 * (D + 4) * 4, "the waves' sums fit where the tiles were");

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ql = lane & 31, half = lane >> 5;
    // Blocks with the most keys first.  Heads that share keys are kv_heads apart, so with 8 key heads (or a multiple) each stays with
    // one XCD's L2.
    const uint32_t per_block = a.heads * a.seqs;
    const int part = blockIdx.x / per_block % a.parts.parts, block = a.blocks - 1 - (int)(blockIdx.x / per_block / a.parts.parts);
    const int kg = wave / (4 / KG);
    const int seq = blockIdx.x % per_block / a.heads, order = blockIdx.x % a.heads;
    const int kv_head = order % a.kv_heads, head = kv_head * (a.heads / a.kv_heads) + order / a.kv_heads;

    const SeqRows qs = seq_rows(a.q_starts, seq, a.q.rows), ks = seq_rows(a.k_starts, seq, a.k.rows);
    const int n = min(qs.count, a.max_q); // its queries that are computed
    if (block * kBlock >= n)
        return;
    const int ahead = ks.count - qs.count; // query i sees keys up to ahead + i
    const int first = block * kBlock + wave % (4 / KG) * 32; // the wave's first query
    const int last_key = ahead + min(block * kBlock + kBlock, n) - 1; // seen by the block
    const int tiles = last_key < 0 ? 0 : last_key / kTokens + 1;
    const int whole = min(max(ahead + block * kBlock + 1, 0) / kTokens, last_key / kTokens); // tiles in front of the last that every query sees in full
    const int tile0 = (int)((int64_t)tiles * part / a.parts.parts), tile1 = (int)((int64_t)tiles * (part + 1) / a.parts.parts);

    uint4 q[D / 16];
    {
        const int64_t row = qs.first + min(first + ql, n - 1);
        const uint16_t *src = (const uint16_t *)a.q.data + row * a.q.row_stride + (int64_t)head * a.q.head_stride + 8 * half;
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
            q[s] = *(const uint4 *)(src + 16 * s);
        // (there before the loop: a wait for them inside it would be one for the tiles that are being loaded)
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
            asm volatile("" : "+v"(q[s].x), "+v"(q[s].y), "+v"(q[s].z), "+v"(q[s].w));
    }
    // Weights are 2^(score - base + lift): base follows the running maximum only when that has left it 2^kSlack behind, which
    // spares nearly every rescaling.  In fp16 the lift leaves weights their normal range down to 2^-20 of the largest one.  bf16 has
    // the exponents of the sums, and its values may stand at their end: there the lift keeps the sum of all weights below 1/2, so
    // that a sum of weights times values stays below the largest of the values.  (At the other end, values below 2^-90 lose digits.)
    constexpr float kSlack = 8;
    const float lift = DTYPE == ABQ_BF16 ? -kSlack - 1 - (float)(32 - __builtin_clz((unsigned)ks.count | 1)) : 6.f;
    const float slack = fminf(kSlack / a.scale_log2, 3e38f); // (finite, so that any score is more than that above none)
    float16v out[D / 32];
    float base = -INFINITY, shift = 0, l = 0, most = -INFINITY; // base: in scores; shift: what is added to scores in powers of two
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            out[d][i] = 0;

    // Loads of a tile: the lane's place in it, in bytes
    const uint16_t *k_src = (const uint16_t *)a.k.data + (int64_t)ks.first * a.k.row_stride + (int64_t)kv_head * a.k.head_stride;
    const uint16_t *v_src = (const uint16_t *)a.v.data + (int64_t)ks.first * a.v.row_stride + (int64_t)kv_head * a.v.head_stride;
    const unsigned lds_at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)&lds[0][0] + wave * kLoads * 1024;
    const int load_row = (wave * kLoads * 64 + lane) / kPieces, load_piece = lane % kPieces;
    constexpr int kRowStep = 64 / kPieces; // rows between a wave's loads
    const uint32_t k_row = load_row * (uint32_t)a.k.row_stride * 2, k_piece = 16 * key_piece<D>(load_row, load_piece);
    const uint32_t v_row = load_row * (uint32_t)a.v.row_stride * 2, v_piece = 16 * value_piece<D>(load_row, load_piece);
    // Load i of a tile's keys (values), into the first or second place for them.  Behind the last tile: the last one again, so that a
    // wave can count what is on its way.
    auto load = [&](bool keys, int tile, int place, int i) {
        tile = min(tile, tile1 - 1);
        const int64_t stride = keys ? a.k.row_stride : a.v.row_stride;
        const uint32_t last = (min(ks.count - tile * kTokens, kTokens) - 1) * (uint32_t)stride * 2;
        // kRowStep rows on, the pieces of keys change places by 4 and those of values not at all; rows behind the last one are
        // copies of it, and never seen
        const uint32_t row = min((keys ? k_row : v_row) + i * kRowStep * (uint32_t)stride * 2, last);
        lds_dma16((keys ? k_src : v_src) + (int64_t)tile * kTokens * stride, row + (keys ? k_piece ^ 64 * i : v_piece),
                        lds_at + ((keys ? 0 : 2) + place) * kTile + i * 1024);
    };
    auto load_keys = [&](int tile, int place) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            load(true, tile, place, i);
    };
    auto load_values = [&](int tile, int place) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            load(false, tile, place, i);
    };
    // All but the newest `newer` loads have arrived, every wave's, and nobody reads what will be overwritten
    auto arrive = [&](auto newer) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(decltype(newer)::value) : "memory");
        __syncthreads();
    };
    typedef std::integral_constant<int, 0> None;
    typedef std::integral_constant<int, kLoads> OneTile;

    typedef float16v Scores[TT];
    // S^T of a tile
    auto scores = [&](int place, Scores &score) {
        const uint8_t *kt = lds[place] + kg * 32 * D * 2;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                score[tt][i] = 0;
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                const int r = 32 * tt + ql;
                const uint4 k = *(const uint4 *)(kt + r * D * 2 + key_piece<D>(r, 2 * s + half) * 16);
                score[tt] = mfma_32x32x16<DTYPE>(k, q[s], score[tt]);
            }
    };
    auto hide = [&](int tile, Scores &score) { // what a query does not see
        const int sees = ahead + first + ql - tile * kTokens - 32 * kg - 4 * half;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                score[tt][i] = 32 * tt + 8 * (i / 4) + i % 4 <= sees ? score[tt][i] : -INFINITY;
    };
    auto find_most = [&](const Scores &score) {
        float x = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                x = fmaxf(x, score[tt][i]);
        most = max_across_halves(x);
    };
    auto follow = [&]() {
        if (__any(most - base > slack)) { // (the difference has no rounding, base + slack would)
            const float to = fmaxf(most, base);
            const float down = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((base - to) * a.scale_log2);
            base = to;
            shift = to == -INFINITY ? 0.f : lift - to * a.scale_log2;
            l *= down;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    out[d][i] *= down;
        }
    };
    // Weights, two at a time
    uint32_t p[2 * TT][4];
    auto weigh = [&](int pair, const Scores &score) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(score[pair / 8][2 * (pair % 8)], a.scale_log2, shift));
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(score[pair / 8][2 * (pair % 8) + 1], a.scale_log2, shift));
        l += x;
        l += y;
        p[pair / 4][pair % 4] = pack16<DTYPE>(x, y);
    };
    // Sixteen tokens at a time: their values, and out^T += V^T P^T
    const int tr = (lane & 15) / 4 + 4 * half, tc = 16 * (lane >> 4 & 1) + 4 * (lane & 3); // the lane's row and element
    uint4 v[2][D / 32];
    auto fetch = [&](int place, int s) {
        const uint8_t *vt = lds[2 + place];
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
            uint2 x[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = 32 * kg + 16 * s + 8 * j + tr, e = 32 * d + tc;
                x[j] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) short4v *)(vt + r * D * 2 + value_piece<D>(r, e / 8) * 16 + e % 8 * 2)));
            }
            v[s & 1][d] = uint4{x[0].x, x[0].y, x[1].x, x[1].y};
        }
    };
    auto gather = [&](int s) {
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
            out[d] = mfma_32x32x16<DTYPE>(v[s & 1][d], uint4{p[s][0], p[s][1], p[s][2], p[s][3]}, out[d]);
    };

    // The scores of a tile are taken while the one before is weighed, and its maximum is found while that one's values are gathered.
    // Loads stand between the products: eight at once would hold a wave up for as long as a quarter of the tile's products take.
    // A tile's keys and values are requested one step before they are needed, keys in a step's first half and values in its second.
    auto step = [&](int tile, auto place, const Scores &score, Scores &next) {
        constexpr int b = decltype(place)::value;
        arrive(OneTile());
        // Sixteen elements at a time: their products, the next ones' keys, and a share of the weights beside each other
        constexpr int kShares = D / 16, kPairs = 8 * TT / kShares, kAhead = 4 / TT - 1; // (keys on their way)
        uint4 k[kAhead + 1][TT];
        auto read_keys = [&](int c) {
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                const int r = 32 * tt + ql;
                k[c % (kAhead + 1)][tt] = *(const uint4 *)(lds[1 - b] + (32 * kg + r) * D * 2 + key_piece<D>(r, 2 * c + half) * 16);
            }
        };
#pragma unroll
        for (int c = 0; c < kAhead; ++c)
            read_keys(c);
        follow();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                next[tt][i] = 0;
#pragma unroll
        for (int c = 0; c < kShares; ++c) {
            if (c + kAhead < kShares)
                read_keys(c + kAhead);
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
                next[tt] = mfma_32x32x16<DTYPE>(k[c % (kAhead + 1)][tt], q[c], next[tt]);
#pragma unroll
            for (int i = 0; i < kPairs; ++i)
                weigh(kPairs * c + i, score);
            if (c % 2 == 1)
                load(true, tile + 2, b, c / 2);
            __builtin_amdgcn_sched_group_barrier(0x100, TT, 0);
#pragma unroll
            for (int i = 0; i < TT; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x402, 7 * 128 / D, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        // (all weights are taken here, not behind the branch)
#pragma unroll
        for (int s = 0; s < 2 * TT; ++s)
            asm volatile("" : "+v"(p[s][0]), "+v"(p[s][1]), "+v"(p[s][2]), "+v"(p[s][3]));
        if (tile + 1 >= whole)
            hide(tile + 1, next);
        arrive(OneTile());
        float x = -INFINITY;
        fetch(b, 0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < 2 * TT; ++s) { // the next sixteen tokens' values and a quarter (half) of the maximum beside the products
            if (s < 2 * TT - 1)
                fetch(b, s + 1);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x = fmaxf(x, next[s / 2][8 * (s % 2) + i]);
            gather(s);
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                if (i * 2 * TT / kLoads == s)
                    load(false, tile + 1, 1 - b, i);
            __builtin_amdgcn_sched_group_barrier(0x100, D / 16, 0);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, 2, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        most = max_across_halves(x);
    };
    if (tile0 < tile1) {
        Scores even, uneven;
        load_keys(tile0, 0);
        arrive(None());
        load_keys(tile0 + 1, 1);
        load_values(tile0, 0);
        scores(0, even);
        if (tile0 >= whole)
            hide(tile0, even);
        find_most(even);
        int tile = tile0;
        for (; tile + 2 < tile1; tile += 2) {
            step(tile, std::integral_constant<int, 0>(), even, uneven);
            step(tile + 1, std::integral_constant<int, 1>(), uneven, even);
        }
        if (tile + 1 < tile1) {
            step(tile, std::integral_constant<int, 0>(), even, uneven);
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
                even[tt] = uneven[tt];
            ++tile;
        }
        arrive(None()); // the last one
        follow();
#pragma unroll
        for (int i = 0; i < 8 * TT; ++i)
            weigh(i, even);
#pragma unroll
        for (int s = 0; s < 2 * TT; ++s) {
            fetch(tile - tile0 & 1, s);
            gather(s);
        }
    }

    // (what the lane is, taken anew: the loop needs every register)
    int none = 0;
    asm volatile("" : "+v"(none));
    const int upper = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, none)) >> 5;

    // A block is done again, step by step, in two cases.
    // A weight of 0 does not keep a value that is not finite out of a product, so one that no query may see can have come into the
    // sums.  Where they are not all finite, and a tile that some query does not see all of holds such values, zeros take their
    // places, and they are added after the product to the queries that see them.
    // Scores from 2^24 powers of two on leave no room for a lift that is added to them: fp32 has steps of 2 and more there.  The base
    // is taken off them first, which has no rounding near it.
    if (whole < tiles) {
        float any = 0;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                any = __builtin_fmaf(out[d][i], 0.f, any);
        const bool found = __any(!(any == 0) || (fabsf(base) < INFINITY && fabsf(base) * a.scale_log2 >= 0x1p24f));
        if (lane == 0)
            odd_values[wave] = found;
        __syncthreads();
        if (odd_values[0] | odd_values[1] | odd_values[2] | odd_values[3]) {
            base = -INFINITY;
            shift = l = 0;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    out[d][i] = 0;
            Scores score;
#pragma unroll 1
            for (int tile = tile0; tile < tile1; ++tile) {
                __syncthreads(); // (nobody reads the tile before)
                load_keys(tile, 0);
                load_values(tile, 0);
                arrive(None());
                if (tile >= whole) {
                    uint4 *piece = (uint4 *)(lds[2] + (wave * 64 + lane) * 16);
#pragma unroll 1
                    for (int i = 0; i < kTile / 4096; ++i) {
                        uint4 w = piece[i * 256];
                        w.x &= ~(not_finite<DTYPE>(w.x) / 0x8000 * 0xffff), w.y &= ~(not_finite<DTYPE>(w.y) / 0x8000 * 0xffff);
                        w.z &= ~(not_finite<DTYPE>(w.z) / 0x8000 * 0xffff), w.w &= ~(not_finite<DTYPE>(w.w) / 0x8000 * 0xffff);
                        piece[i * 256] = w;
                    }
                    __syncthreads();
                }
                scores(0, score);
                if (tile >= whole)
                    hide(tile, score);
                find_most(score);
                follow();
                shift = lift;
                {
                    const float from = fabsf(base) < INFINITY ? base : 0.f;
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            score[tt][i] -= from;
                }
#pragma unroll
                for (int i = 0; i < 8 * TT; ++i)
                    weigh(i, score);
#pragma unroll
                for (int s = 0; s < 2 * TT; ++s) {
                    fetch(0, s);
                    gather(s);
                }
                if (tile < whole)
                    continue;
#pragma unroll 1
                for (int tok = 32 * kg; tok < min(32 * kg + 32 * TT, ks.count - tile * kTokens); ++tok) {
                    const uint16_t *src = v_src + (int64_t)(tile * kTokens + tok) * a.v.row_stride + 4 * upper;
                    const int i = tok % 32 / 8 * 4 + tok % 4;
                    uint32_t pair = 0;
#pragma unroll
                    for (int j = 0; j < 8 * TT; ++j)
                        pair = (tok / 32 - kg) * 8 + i / 2 == j ? p[j / 4][j % 4] : pair;
                    pair = __shfl(pair, ql + 32 * (tok / 4 % 2));
                    const float w = value16<DTYPE>(i & 1 ? pair >> 16 : pair);
                    const bool seen = tile * kTokens + tok - ahead - first <= ql;
#pragma unroll
                    for (int d = 0; d < D / 32; ++d) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint2 four = *(const uint2 *)(src + 32 * d + 8 * j);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float x = value16<DTYPE>((e < 2 ? four.x : four.y) >> (16 * (e & 1)));
                                out[d][4 * j + e] = __builtin_fmaf(w, seen && !(fabsf(x) < INFINITY) ? x : 0.f, out[d][4 * j + e]);
                            }
                        }
                        asm volatile("" ::: "memory"); // (a few loads at a time)
                    }
                }
            }
            shift = base == -INFINITY ? 0.f : lift - base * a.scale_log2;
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // (nothing may arrive in LDS that is another's, or holds sums)

    // the sums of the waves with the other tokens
    if constexpr (KG == 2) {
        float *sums = (float *)&lds[0][0];
        __shared__ float other[2][64];
        const int r = wave % 2 * 32 + ql;
        __syncthreads();
        if (kg == 1) {
            l = sum_across_halves(l);
            if (upper == 0) {
                other[0][r] = base;
                other[1][r] = l;
            }
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *(float4 *)&sums[r * (D + 4) + 32 * d + 8 * j + 4 * upper] = float4{out[d][4 * j], out[d][4 * j + 1], out[d][4 * j + 2], out[d][4 * j + 3]};
        }
        __syncthreads();
        if (kg == 1)
            return;
        const float b = other[0][r], to = fmaxf(b, base);
        const float mine = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((base - to) * a.scale_log2);
        const float theirs = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((b - to) * a.scale_log2);
        base = to;
        shift = to == -INFINITY ? 0.f : lift - to * a.scale_log2;
        l = l * mine + (upper ? 0.f : other[1][r] * theirs);
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int j = 0; j < 16; ++j)
                out[d][j] = out[d][j] * mine + sums[r * (D + 4) + 32 * d + 8 * (j / 4) + 4 * upper + j % 4] * theirs;
    }

    const float total = sum_across_halves(l);
    const int i = first + ql;
    if (a.parts.parts > 1) {
        if (i < n) {
            const int64_t at = ((int64_t)(qs.first + i) * a.heads + head) * a.parts.parts + part;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *(float4 *)(a.parts.sums + at * D + 32 * d + 8 * j + 4 * upper) = float4{out[d][4 * j], out[d][4 * j + 1], out[d][4 * j + 2], out[d][4 * j + 3]};
            if (upper == 0)
                a.parts.stats[at] = float2{base == -INFINITY ? -INFINITY : -shift, total};
        }
        return;
    }
    float f = total > 0 ? 1.f / total : total; // (a sum that is not a number stays one)
    // (a finite result becomes the type's largest at most: saturated16; fp16 has a bit of the wave's mode for it, which lets infinities be)
    if constexpr (DTYPE == ABQ_F16) {
        __builtin_amdgcn_s_setreg(1 | 23 << 6, 1); // MODE.FP16_OVFL
        asm volatile("" : "+v"(f));                // (the conversions come behind it)
    } else {
        float far = 0;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int j = 0; j < 16; ++j)
                far = fmaxf(far, fabsf(out[d][j]));
        if (__any(far * f > largest16<DTYPE>())) {
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    out[d][j] = saturated16<DTYPE>(out[d][j] * f);
            f = 1.f;
        }
    }
    uint16_t *to = (uint16_t *)a.out.data + (int64_t)(qs.first + i) * a.out.row_stride + (int64_t)head * a.out.head_stride;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            // elements 8 x + 4 h .. + 3 of the lanes h = 0, 1: eight neighbours per lane after an exchange
            uint32_t x[2][2];
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    x[y][e] = pack16<DTYPE>(out[d][8 * j + 4 * y + 2 * e] * f, out[d][8 * j + 4 * y + 2 * e + 1] * f);
            const auto r0 = __builtin_amdgcn_permlane32_swap(x[0][0], x[1][0], false, false);
            const auto r1 = __builtin_amdgcn_permlane32_swap(x[0][1], x[1][1], false, false);
            if (i < n)
                *(uint4 *)(to + 32 * d + 16 * j + 8 * upper) = uint4{r0[0], r1[0], r0[1], r1[1]};
        }
}

} // namespace

void plan_attn_prompt(abq_attn_state *st, int most_parts)
{
    const int64_t each = (int64_t)st->heads * st->seqs;
    // A compute unit holds two workgroups, so 512 run beside each other.  With fewer blocks of 128 queries, blocks of 64 whose
    // waves share the tokens (1024 tokens, heads of 128, fp16: 32 heads 23.6 -> 19.9 us, 8 heads 21.3 -> 15.5; 64 heads, which
    // fill the chip, 29.5 -> 34) ...
    st->block_rows = ((int64_t)st->max_q + 127) / 128 * each >= 512 ? 128 : 64;
    // ... and where those leave room as well, parts of the keys: one workgroup per compute unit, or two with heads of 64.  A part
    // saves its share of the steps, 0.6 us (0.5) each; the parts' results cost a launch, 3 us, and their way through memory.
    //   us in parts                               1     2     4     8    16    32
    //   64 queries behind 8128, 4 heads of 128   78    46    28    19    15    14   (taken: 32)
    //   the same, 16 heads                       79    47    29    20    20    24   (16)
    //   512 behind 3584, 16 heads of 128         44    34    34    44    71         (2)
    //   1024 alone, 8 heads of 128               15    17    18                     (1)
    //   333 behind 7000, 8 heads of 64           62    38    24    20    22    25   (10)
    const int64_t groups = ((int64_t)st->max_q + st->block_rows - 1) / st->block_rows * each;
    const double steps = ((int64_t)st->max_k + kTokens - 1) / kTokens, step_us = st->head_dim == 64 ? 0.5 : 0.6;
    const double result_us = (double)st->q.rows * st->heads * st->head_dim * 8 / 4e6;
    int64_t most = (st->head_dim == 64 ? 512 : 256) / groups, parts = 1;
    most = most < steps / 4 ? most : (int64_t)(steps / 4);
    most = most < most_parts ? most : most_parts;
    double least = steps * step_us;
    for (int64_t p = 2; p <= most; ++p) {
        const double us = steps / p * step_us + 3 + p * result_us;
        if (us < least) {
            least = us;
            parts = p;
        }
    }
    st->parts = (int)parts;
}

#define ABQ_PROMPT(T, D_, KG) hipLaunchKernelGGL((attn_prompt_kernel<T, D_, KG>), grid, dim3(256), 0, stream, a)
#define ABQ_PROMPT_DIM(T)                    \
    do {                                     \
        if (st.head_dim == 64) {             \
            if (st.block_rows == 128)        \
                ABQ_PROMPT(T, 64, 1);        \
            else                             \
                ABQ_PROMPT(T, 64, 2);        \
        } else if (st.block_rows == 128)     \
            ABQ_PROMPT(T, 128, 1);           \
        else                                 \
            ABQ_PROMPT(T, 128, 2);           \
    } while (0)

hipError_t launch_attn_prompt(const abq_attn_state &st, hipStream_t stream)
{
    PromptArgs a;
    a.q = st.q;
    a.k = st.k;
    a.v = st.v;
    a.out = st.out;
    a.q_starts = st.q_starts;
    a.k_starts = st.k_starts;
    a.heads = st.heads;
    a.kv_heads = st.kv_heads;
    a.seqs = st.seqs;
    a.max_q = st.max_q;
    a.blocks = (st.max_q + st.block_rows - 1) / st.block_rows;
    a.scale_log2 = st.scale * kLog2e;
    a.parts = attn_parts(st);
    const dim3 grid((unsigned)((int64_t)a.blocks * st.heads * st.seqs * st.parts));
    if (st.dtype == ABQ_BF16)
        ABQ_PROMPT_DIM(ABQ_BF16);
    else
        ABQ_PROMPT_DIM(ABQ_F16);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess || st.parts < 2 ? e : launch_attn_join(st, stream);
}

} // namespace abq
