// Attention of drafted tokens (ordinary decoding: one) over the quantised, paged cache.
//
// The query heads that share a key head and the drafts of a sequence are the rows of one product: row r is draft r / group,
// head r % group.  With u the stored codes, s and z a token's scale and zero point, and everything in powers of two,
//     score[t][r] = s_k[t] (u_k[t] . q[r] - z_k[t] sum(q[r])) scale log2(e)
//     w[t][r]     = 2^(score[t][r] + log2(s_v[t]) - max_t(same))
//     out[r]      = (sum_t w[t][r] u_v[t] - sum_t w[t][r] z_v[t]) / sum_t (w[t][r] / s_v[t])
// so codes enter the matrix cores as the whole numbers they are, exact in fp16, and are never scaled one by one: a code costs
// one half of a byte permute (or mask) and one half of a packed add.  Folding s_v into the exponent keeps the largest weight at
// 1 whatever the scales are, so that weights rounded to fp16 (11 bits; the one rounding of the sum, as large as that of the
// result) do not run into its subnormals.  Queries in bf16 become fp16 after a division of each row by a power of two: elements
// down to 2^-31 of the row's largest keep all their bits, those below 2^-39 of it become 0, which a 32-bit sum beside the largest
// one's term would lose as well.  Sums of weights are taken before they are rounded, those of weights times zero points behind it.
//
// Both products are taken transposed, scores^T = K q^T and out^T = V^T w^T (16 x 16 x 32 MFMA), because the result of the
// first then lies in the registers as the second wants it: lane (r, g) gets the scores of row r for tokens 4 g .. 4 g + 3, and
// gives the weights of the tokens 4 g .. 4 g + 3 of both halves of a 32-token step as its eight.  The cache keeps four tokens'
// values beside each other for the same reason.  A wave goes from global memory to registers in 16-byte loads and needs no
// LDS until its tokens are done.
//
// A sequence's tokens are split over workgroups (parts) until the chip is covered, and inside one over its waves, step by
// step; the waves' results are joined in LDS, the parts' by a second launch.
//
// Up to 16 rows, bound by the cache's bytes: one query for each of 32 heads on 16 x 1024 tokens of 8 bits, 29 us for 138 MB,
// 4.8 TB/s of the 5.1 that a copy reaches; four waves per SIMD cover each other's loads, so none keeps a second buffer.  With more
// rows a step's vector work (400 operations beside 32 MFMA: codes to fp16, factors, exponentials) and the loads share the time:
// two waves per SIMD, each with a step under way while it works at another.  20 rows on 48 ragged contexts, 630 MB: 148 us,
// 4.3 TB/s; 108 rows on 3 x 5500 tokens of 4 bits, 28 us, bound by that work and, at 9 steps a wave, by its start and end.
#include "abq_attn.h"

namespace abq {

namespace {

struct TreeArgs {
    abq_kv_cache c;
    abq_rows q, out;
    const int32_t *page_table, *context, *q_starts;
    const uint64_t *mask;
    int heads, group, seqs, max_q, max_pages, row_blocks, dtype;
    int page_shift;
    float scale_log2;
    AttnParts parts;
};

constexpr int kStep = 32; // tokens of a wave's step
constexpr int tree_waves(int row_tiles) { return row_tiles == 1 ? 8 : 4; }

__device__ __forceinline__ half2v half2_bits(uint32_t w) { return __builtin_bit_cast(half2v, w); }
__device__ __forceinline__ uint32_t bits(half2v h) { return __builtin_bit_cast(uint32_t, h); }

// What a wave reads for one step.  K: per 16 tokens, the lane's bytes of its token's row.  V: per half, four tokens' words.
template <int BITS, bool ASYM, int D> struct Step {
    // words of a lane per 16 tokens, of keys and of values
    static constexpr int kWords = D * BITS / 128;
    static constexpr int kLoad = kWords < 4 ? kWords : 4; // words per load
    uint32_t k[2][kWords], v[2][kWords];
    float ks, vs, kz, vz; // of one token: lanes t = 4 h + i of the quarter g have token 4 g + i of half h, lanes 8 + t the same
};

template <int N> __device__ __forceinline__ void load_words(uint32_t *to, const void *from)
{
    if constexpr (N == 4) {
        const uint4 w = *(const uint4 *)from;
        to[0] = w.x, to[1] = w.y, to[2] = w.z, to[3] = w.w;
    } else {
        const uint2 w = *(const uint2 *)from;
        to[0] = w.x, to[1] = w.y;
    }
}
// What lane K of the lane's row of sixteen has
template <int K> __device__ __forceinline__ uint32_t of_lane(uint32_t x)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x150 + K, 0xf, 0xf, true);
}
template <int K> __device__ __forceinline__ float of_lane(float x)
{
    return __builtin_bit_cast(float, of_lane<K>(__builtin_bit_cast(uint32_t, x)));
}

// `seen`: bit h is cleared if half h lies on a page outside the cache
template <int BITS, bool ASYM, int D>
__device__ __forceinline__ void load_step(Step<BITS, ASYM, D> &s, const TreeArgs &a, const int32_t *pages, int last_page, int head, int at, int lane,
                                          uint32_t *seen)
{
    using S = Step<BITS, ASYM, D>;
    constexpr int R = D * BITS / 8;
    const int t = lane & 15, g = lane >> 4;
    int64_t rows[2];
    *seen = 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int pos = at + 16 * h;
        int page = pages[min(pos >> a.page_shift, last_page)];
        if ((uint32_t)page >= (uint32_t)a.c.num_pages) {
            page = 0;
            *seen &= ~(1u << h);
        }
        const int in_page = pos & (a.c.page_size - 1);
        const int64_t row = ((int64_t)page * a.c.kv_heads + head) * a.c.page_size;
        const uint8_t *k = (const uint8_t *)a.c.k_codes + (row + in_page + t) * R;
        const uint8_t *v = (const uint8_t *)a.c.v_codes + (row + in_page + 4 * g) * R;
#pragma unroll
        for (int l = 0; l < S::kWords / S::kLoad; ++l) {
            load_words<S::kLoad>(&s.k[h][l * S::kLoad], k + l * 64 + g * 4 * S::kLoad);
            load_words<S::kLoad>(&s.v[h][l * S::kLoad], v + l * 256 + t * 4 * S::kLoad);
        }
        rows[h] = (ASYM ? 2 : 1) * row + in_page;
    }
    const int64_t at_scale = (t & 4 ? rows[1] : rows[0]) + 4 * g + (t & 3);
    s.ks = a.c.k_scales[at_scale];
    s.vs = a.c.v_scales[at_scale];
    if (ASYM) {
        s.kz = a.c.k_scales[at_scale + a.c.page_size];
        s.vz = a.c.v_scales[at_scale + a.c.page_size];
    }
}

// Codes to fp16: 1024 + u is the number 0x6400 | u.  The constants stand in registers of their own, one scalar and one vector, for
// an operation to take both.
struct Magic {
    uint32_t bytes, halves; // 0x64 in every byte, 0x6400 in both halves
};
__device__ __forceinline__ Magic magic()
{
    Magic m = {0x64646464u, 0x64006400u};
    asm("" : "+v"(m.bytes), "+v"(m.halves));
    return m;
}
// Four codes of a word less half the range, in two pairs
__device__ __forceinline__ void four_codes(const Magic &m, uint32_t w, uint32_t *lo, uint32_t *hi)
{
    const half2v off = {(_Float16)1152, (_Float16)1152};
    *lo = bits(half2_bits(__builtin_amdgcn_perm(m.bytes, w, 0x04010400u)) - off);
    *hi = bits(half2_bits(__builtin_amdgcn_perm(m.bytes, w, 0x04030402u)) - off);
}
// Eight 4-bit codes of a word: nibbles (0, 4), (1, 5), (2, 6), (3, 7).  A nibble in bits 4 - 7 stands for 16 times its value.
__device__ __forceinline__ void eight_codes(const Magic &m, uint32_t w, uint32_t *out)
{
    const half2v off = {(_Float16)1032, (_Float16)1032}, part = {(_Float16)0.0625f, (_Float16)0.0625f}, off16 = {(_Float16)72, (_Float16)72};
    const uint32_t w8 = w >> 8;
    out[0] = bits(half2_bits((w & 0x000f000fu) | m.halves) - off);
    out[1] = bits(half2_bits((w & 0x00f000f0u) | m.halves) * part - off16);
    out[2] = bits(half2_bits((w8 & 0x000f000fu) | m.halves) - off);
    out[3] = bits(half2_bits((w8 & 0x00f000f0u) | m.halves) * part - off16);
}

// (score * k_factor + k_offset * qsum) * factor + v_log of token K of the lane's eight and of those behind it.  The row's power of
// two comes last: in units of codes a score that fp32 holds may be beyond it.
template <bool ASYM, int RT, int K>
__device__ __forceinline__ void exponents(float (&score)[RT][2][4], float k_factor, float k_offset, float v_log, const float (&qsum)[RT],
                                          const float (&factor)[RT])
{
    if constexpr (K < 8) {
        const float f = of_lane<K>(k_factor), v = of_lane<K>(v_log), o = ASYM ? of_lane<K>(k_offset) : 0.f;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float x = score[rt][K / 4][K % 4] * f;
            score[rt][K / 4][K % 4] = __builtin_fmaf(ASYM ? __builtin_fmaf(o, qsum[rt], x) : x, factor[rt], v);
        }
        exponents<ASYM, RT, K + 1>(score, k_factor, k_offset, v_log, qsum, factor);
    }
}
// sum + the tokens' weights times their v
template <int K> __device__ __forceinline__ float weighted_sum(const float (&w)[2][4], float v, float sum)
{
    if constexpr (K < 8)
        return weighted_sum<K + 1>(w, v, __builtin_fmaf(of_lane<K>(v), w[K / 4][K % 4], sum));
    return sum;
}
template <int K> __device__ __forceinline__ float pair_sum(const uint32_t (&w)[4], uint32_t v, float sum)
{
    if constexpr (K < 4)
        return pair_sum<K + 1>(w, v, __builtin_amdgcn_fdot2(half2_bits(w[K]), half2_bits(of_lane<2 * K>(v)), sum, false));
    return sum;
}

__device__ __forceinline__ half8v half8_bits(const uint32_t *w)
{
    const uint4 x = {w[0], w[1], w[2], w[3]};
    return __builtin_bit_cast(half8v, x);
}

// A lane's 8-element pieces of the queries: piece ks of D / 32, in the order of the keys' bytes
template <int BITS, int D> __device__ __forceinline__ int query_offset(int ks, int g)
{
    constexpr int kPieces = BITS == 8 ? 2 : (D == 128 ? 4 : 2); // pieces per load of a lane
    return (ks / kPieces) * (32 * kPieces) + g * 8 * kPieces + (ks % kPieces) * 8;
}

template <int BITS, bool ASYM, int D, int RT> __global__ __launch_bounds__(64 * tree_waves(RT), RT == 1 ? 4 : 2) void attn_tree_kernel(TreeArgs a)
{
    using S = Step<BITS, ASYM, D>;
    constexpr int kWaves = tree_waves(RT);
    constexpr int kTiles = D / 16; // 16 x 16 tiles of out^T
    constexpr int kPad = D + 4;
    __shared__ __align__(16) float sums[kWaves][16][kPad];
    __shared__ float stat_m[kWaves][16 * RT], stat_l[kWaves][16 * RT], stat_z[kWaves][16 * RT];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = lane & 15, g = lane >> 4;
    // Workgroups go round the eight XCDs: those that read the same tokens (other rows of them) are eight apart, on one L2.
    const uint32_t round = 8 * a.row_blocks, in_round = blockIdx.x % round;
    const uint32_t unit = blockIdx.x / round * 8 + in_round % 8;
    const int row_block = in_round / 8;
    if (unit >= (uint32_t)a.seqs * a.c.kv_heads * a.parts.parts)
        return;
    const int part = unit % a.parts.parts, head = unit / a.parts.parts % a.c.kv_heads, seq = unit / a.parts.parts / a.c.kv_heads;

    const SeqRows own = seq_rows(a.q_starts, seq, a.q.rows);
    const int n = min(own.count, 64); // drafts that can be seen, of which max_q are computed
    const int rows = min(n, a.max_q) * a.group, row0 = row_block * 16 * RT;
    if (row0 >= rows)
        return;
    const int64_t places = (int64_t)a.max_pages << a.page_shift;
    const int context = (int)min((int64_t)max(a.context[seq], 0), places);
    const int len = (int)min((int64_t)context + n, places);
    const int32_t *pages = a.page_table + (int64_t)seq * a.max_pages;
    const int last_page = (len - 1) >> a.page_shift; // (len is 0 only without steps)

    // the queries as the products take them, the power of two that they were divided by, and their sums
    half8v q[RT][D / 32];
    float factor[RT], qsum[RT];
    uint64_t sees[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int row = min(row0 + 16 * rt + t, rows - 1), draft = row / a.group;
        const uint16_t *src = (const uint16_t *)a.q.data + (int64_t)(own.first + draft) * a.q.row_stride + (int64_t)(head * a.group + row % a.group) * a.q.head_stride;
        sees[rt] = a.mask ? a.mask[own.first + draft] : ~0ull >> (63 - draft);
        factor[rt] = 1.f;
        float sum = 0;
        uint4 w[D / 32];
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks)
            w[ks] = *(const uint4 *)(src + query_offset<BITS, D>(ks, g));
        if (a.dtype == ABQ_BF16) {
            float most = 0;
#pragma unroll
            for (int ks = 0; ks < D / 32; ++ks) {
                const uint32_t x[4] = {w[ks].x, w[ks].y, w[ks].z, w[ks].w};
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    most = fmaxf(most, fabsf(bf16_value(x[i / 2] >> (16 * (i & 1)) & 0xffff)));
            }
            most = max_across_quarters(most);
            // the largest becomes [2^14, 2^15), if 2^126 gets it there
            const int e = most > 0 && most < INFINITY ? min(14 + 127 - (int)(__builtin_bit_cast(uint32_t, most) >> 23), 126) : 0;
            const float up = __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
            factor[rt] = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
#pragma unroll
            for (int ks = 0; ks < D / 32; ++ks) {
                const uint32_t x[4] = {w[ks].x, w[ks].y, w[ks].z, w[ks].w};
                uint32_t y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    y[i] = pack16<ABQ_F16>(bf16_value(x[i] & 0xffff) * up, bf16_value(x[i] >> 16) * up);
                q[rt][ks] = half8_bits(y);
            }
        } else
#pragma unroll
            for (int ks = 0; ks < D / 32; ++ks)
                q[rt][ks] = __builtin_bit_cast(half8v, w[ks]);
        if (ASYM)
#pragma unroll
            for (int ks = 0; ks < D / 32; ++ks)
#pragma unroll
                for (int i = 0; i < 8; i += 2)
                    sum = __builtin_amdgcn_fdot2(half2v{q[rt][ks][i], q[rt][ks][i + 1]}, half2v{(_Float16)1, (_Float16)1}, sum, false);
        qsum[rt] = ASYM ? sum_across_quarters(sum) : 0;
    }

    float4v out[RT][kTiles];
    // Weights are 2^(exponent - base + kLift): base follows the running maximum only when that has left it 2^kSlack behind, which
    // spares nearly every rescaling, and the lift leaves fp16 its normal range down to 2^-24 of the largest weight.
    constexpr float kSlack = 5, kLift = 10;
    float base[RT], shift[RT], l[RT], z[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        base[rt] = -INFINITY;
        shift[rt] = l[rt] = z[rt] = 0;
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
            out[rt][i] = float4v{0, 0, 0, 0};
    }

    const int steps = (len + kStep - 1) / kStep;
    const int step0 = (int)((int64_t)steps * part / a.parts.parts) + wave, step1 = (int)((int64_t)steps * (part + 1) / a.parts.parts);
    const Magic mg = magic();
    auto weigh_step = [&](S &s, int step, uint32_t seen) {
        // scores
        float score[RT][2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float4v acc[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                acc[rt] = float4v{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < D / 32; ++ks) {
                uint32_t w[4];
                if (BITS == 8) {
                    four_codes(mg, s.k[h][2 * ks], &w[0], &w[1]);
                    four_codes(mg, s.k[h][2 * ks + 1], &w[2], &w[3]);
                } else
                    eight_codes(mg, s.k[h][ks], w);
                const half8v k = half8_bits(w);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[rt][ks], acc[rt], 0, 0, 0);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    score[rt][h][i] = acc[rt][i];
        }
        // The lane's one token: factor and offset of the scores, logarithm and reciprocal of the value scale.  (Codes are less half
        // their range here, and so are zero points.)  What no row sees holds anything, and is replaced.
        const int at = step * kStep;
        const bool some = at + kStep > context || seen != 3; // (some row does not see some token of the step)
        if (some) {
            const int h = t >> 2 & 1;
            const bool there = at + 16 * h + 4 * g + (t & 3) < len && (seen >> h & 1);
            s.ks = there ? s.ks : 0.f;
            s.vs = there ? s.vs : 1.f;
            if (ASYM) {
                s.kz = there ? s.kz : 0.f;
                s.vz = there ? s.vz : 0.f;
            }
        }
        constexpr float kHalf = (float)(1 << (BITS - 1));
        const float k_factor = s.ks * a.scale_log2, k_offset = ASYM ? k_factor * (kHalf - s.kz) : 0.f;
        const float v_log = __builtin_amdgcn_logf(s.vs), v_recip = __builtin_amdgcn_rcpf(s.vs);
        // Zero points as fp16 pairs: whole numbers beyond fp16's 2048 in two parts, multiples of 2048 and the rest
        uint32_t z_low = 0, z_high = 0;
        bool high = false;
        if constexpr (ASYM) {
            const float x = s.vz - kHalf, xh = rintf(x * (1.f / 2048)) * 2048.f;
            const float y = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0xb1, 0xf, 0xf, true)); // of lane t ^ 1
            const float yh = rintf(y * (1.f / 2048)) * 2048.f;
            z_low = pack16<ABQ_F16>(x - xh, y - yh); // (used of even lanes)
            z_high = pack16<ABQ_F16>(xh, yh);
            high = __any(xh != 0);
        }
        exponents<ASYM, RT, 0>(score, k_factor, k_offset, v_log, qsum, factor);
        if (some)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int pos = at + 16 * h + 4 * g + i;
                    const bool there = pos < len && (seen >> h & 1);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        score[rt][h][i] = there && (pos < context || (sees[rt] >> ((pos - context) & 63) & 1)) ? score[rt][h][i] : -INFINITY;
                }
        // weights
        half8v w[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float most = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    most = fmaxf(most, score[rt][h][i]);
            most = max_across_quarters(most);
            if (__any(most - base[rt] > kSlack)) { // (the difference has no rounding)
                const float to = fmaxf(most, base[rt]);
                const float down = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(base[rt] - to);
                base[rt] = to;
                // (from 2^24 on the lift is rounded to steps of 2 and more: never to more than it is)
                const float lifted = kLift - to;
                shift[rt] = to == -INFINITY ? 0.f : lifted + to > kLift ? -to : lifted;
                l[rt] *= down;
                z[rt] *= down;
#pragma unroll
                for (int i = 0; i < kTiles; ++i)
                    out[rt][i] *= down;
            }
            uint32_t pair[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    score[rt][h][i] = __builtin_amdgcn_exp2f(score[rt][h][i] + shift[rt]);
                pair[2 * h] = pack16<ABQ_F16>(score[rt][h][0], score[rt][h][1]);
                pair[2 * h + 1] = pack16<ABQ_F16>(score[rt][h][2], score[rt][h][3]);
            }
            l[rt] = weighted_sum<0>(score[rt], v_recip, l[rt]);
            if constexpr (ASYM) { // with the weights as they are multiplied, so that the two sums' difference has no error of its own
                z[rt] = pair_sum<0>(pair, z_low, z[rt]);
                if (high)
                    z[rt] = pair_sum<0>(pair, z_high, z[rt]);
            }
            w[rt] = half8_bits(pair);
        }
        // out^T += V^T w^T.  8 bits: word j of load i is element 64 i + 4 t + j; 4 bits: two elements, D / 2 apart
#pragma unroll
        for (int j = 0; j < S::kWords; ++j) {
            if (BITS == 8) {
                uint32_t x[4];
                four_codes(mg, s.v[0][j], &x[0], &x[1]);
                four_codes(mg, s.v[1][j], &x[2], &x[3]);
                const half8v v = half8_bits(x);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    out[rt][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w[rt], out[rt][j], 0, 0, 0);
            } else {
                uint32_t x[4], y[4];
                eight_codes(mg, s.v[0][j], x);
                eight_codes(mg, s.v[1][j], y);
                const uint32_t low[4] = {x[0], x[2], y[0], y[2]}, high[4] = {x[1], x[3], y[1], y[3]};
                const half8v v0 = half8_bits(low), v1 = half8_bits(high);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    out[rt][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, w[rt], out[rt][j], 0, 0, 0);
                    out[rt][j + S::kWords] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, w[rt], out[rt][j + S::kWords], 0, 0, 0);
                }
            }
        }
    };
    // One row tile leaves registers for four waves per SIMD, which cover each other's loads; with more, a wave loads a step ahead.
    // Eight waves in a workgroup keep them there where there are few workgroups (of four and of eight: 32768 tokens, 8 heads 25 and 20
    // us, 20 x 700 tokens 11.3 and 10.2, 16 x 1024 of 32 heads 29 either way; sixteen 20, 10.6, 34).
    if constexpr (RT == 1) {
        for (int step = step0; step < step1; step += kWaves) {
            S s;
            uint32_t seen;
            load_step<BITS, ASYM, D>(s, a, pages, last_page, head, step * kStep, lane, &seen);
            weigh_step(s, step, seen);
        }
    } else {
        S s[2];
        uint32_t seen[2];
        if (step0 < step1)
            load_step<BITS, ASYM, D>(s[0], a, pages, last_page, head, step0 * kStep, lane, &seen[0]);
        for (int step = step0; step < step1; step += 2 * kWaves) {
            if (step + kWaves < step1)
                load_step<BITS, ASYM, D>(s[1], a, pages, last_page, head, (step + kWaves) * kStep, lane, &seen[1]);
            weigh_step(s[0], step, seen[0]);
            if (step + kWaves >= step1)
                break;
            if (step + 2 * kWaves < step1)
                load_step<BITS, ASYM, D>(s[0], a, pages, last_page, head, (step + 2 * kWaves) * kStep, lane, &seen[0]);
            weigh_step(s[1], step + kWaves, seen[1]);
        }
    }

    // the waves' results joined
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float total = sum_across_quarters(l[rt]), zeros = ASYM ? sum_across_quarters(z[rt]) : 0;
        if (g == 0) {
            stat_m[wave][16 * rt + t] = base[rt] == -INFINITY ? -INFINITY : -shift[rt];
            stat_l[wave][16 * rt + t] = total;
            stat_z[wave][16 * rt + t] = zeros;
        }
    }
    constexpr int kSpan = BITS == 8 ? 4 : S::kWords; // neighbouring elements that tiles j, j + 1 .. hold
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kTiles && row0 + 16 * rt + t < rows; j += kSpan)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < kSpan; ++e)
                    sums[wave][t][j * 16 + (4 * g + i) * kSpan + e] = out[rt][j + e][i];
        __syncthreads();
        constexpr int kEach = D / 16;
        const int r = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * kEach, row = row0 + 16 * rt + r;
        if (r >= 16 || row >= rows)
            continue;
        float most = -INFINITY, total = 0, acc[kEach];
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
            most = fmaxf(most, stat_m[w][16 * rt + r]);
        const float from = most == -INFINITY ? 0.f : most;
#pragma unroll
        for (int e = 0; e < kEach; ++e)
            acc[e] = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(stat_m[w][16 * rt + r] - from);
            total += f * stat_l[w][16 * rt + r];
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                acc[e] += f * (sums[w][r][d0 + e] - (ASYM ? stat_z[w][16 * rt + r] : 0.f));
        }
        const int64_t q_row = own.first + row / a.group;
        const int q_head = head * a.group + row % a.group;
        if (a.parts.parts > 1) {
            const int64_t at = (q_row * a.heads + q_head) * a.parts.parts + part;
            float *to = a.parts.sums + at * D + d0;
#pragma unroll
            for (int e = 0; e < kEach; e += 4)
                *(float4 *)(to + e) = float4{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
            if ((threadIdx.x & 15) == 0)
                a.parts.stats[at] = float2{most, total};
        } else {
            const float f = total > 0 ? 1.f / total : total; // (a sum that is not a number stays one)
            uint16_t *to = (uint16_t *)a.out.data + q_row * a.out.row_stride + (int64_t)q_head * a.out.head_stride + d0;
            uint32_t x[kEach / 2];
#pragma unroll
            for (int e = 0; e < kEach / 2; ++e)
                x[e] = a.dtype == ABQ_BF16 ? pack16_saturated<ABQ_BF16>(acc[2 * e] * f, acc[2 * e + 1] * f)
                                           : pack16_saturated<ABQ_F16>(acc[2 * e] * f, acc[2 * e + 1] * f);
            if constexpr (kEach == 8)
                *(uint4 *)to = uint4{x[0], x[1], x[2], x[3]};
            else
                *(uint2 *)to = uint2{x[0], x[1]};
        }
    }
}

// The parts of one query row and head per wave
struct JoinArgs {
    abq_rows out;
    AttnParts parts;
    const int32_t *q_starts;
    int seqs, max_q, heads, dtype;
};

template <int D> __global__ __launch_bounds__(256) void attn_join_kernel(JoinArgs a)
{
    const int lane = threadIdx.x & 63;
    const uint32_t unit = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int head = unit % a.heads, draft = unit / a.heads % a.max_q, seq = unit / a.heads / a.max_q;
    if (seq >= a.seqs)
        return;
    const SeqRows own = seq_rows(a.q_starts, seq, a.out.rows);
    if (draft >= own.count)
        return;
    const int64_t row = own.first + draft, at = (row * a.heads + head) * a.parts.parts;
    // D / 4 lanes a part, four elements each, so 2 (4) parts at a time, each with a maximum of its own
    constexpr int kLanes = D / 4, kSide = 64 / kLanes;
    const int e0 = lane % kLanes * 4;
    float most = -INFINITY, total = 0, acc[4] = {};
#pragma unroll 4
    for (int p = lane / kLanes; p < a.parts.parts; p += kSide) {
        const float2 st = a.parts.stats[at + p];
        const float4 x = *(const float4 *)(a.parts.sums + (at + p) * D + e0);
        const float to = fmaxf(most, st.x), base = to == -INFINITY ? 0.f : to;
        const float f = __builtin_amdgcn_exp2f(most - base), g = __builtin_amdgcn_exp2f(st.x - base);
        most = to;
        total = total * f + st.y * g;
        acc[0] = acc[0] * f + x.x * g, acc[1] = acc[1] * f + x.y * g, acc[2] = acc[2] * f + x.z * g, acc[3] = acc[3] * f + x.w * g;
    }
#pragma unroll
    for (int o = kLanes; o < 64; o *= 2) {
        const float other = __shfl_xor(most, o), to = fmaxf(most, other), base = to == -INFINITY ? 0.f : to;
        const float f = __builtin_amdgcn_exp2f(most - base), g = __builtin_amdgcn_exp2f(other - base);
        most = to;
        total = total * f + __shfl_xor(total, o) * g;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            acc[e] = acc[e] * f + __shfl_xor(acc[e], o) * g;
    }
    const float f = total > 0 ? 1.f / total : total;
    uint16_t *to = (uint16_t *)a.out.data + row * a.out.row_stride + (int64_t)head * a.out.head_stride + e0;
    if (lane < kLanes)
        *(uint2 *)to = a.dtype == ABQ_BF16 ? uint2{pack16_saturated<ABQ_BF16>(acc[0] * f, acc[1] * f), pack16_saturated<ABQ_BF16>(acc[2] * f, acc[3] * f)}
                                           : uint2{pack16_saturated<ABQ_F16>(acc[0] * f, acc[1] * f), pack16_saturated<ABQ_F16>(acc[2] * f, acc[3] * f)};
}

} // namespace

hipError_t launch_attn_join(const abq_attn_state &st, hipStream_t stream)
{
    const JoinArgs a = {st.out, attn_parts(st), st.q_starts, st.seqs, st.max_q, st.heads, st.dtype};
    const dim3 grid((unsigned)(((int64_t)st.seqs * st.max_q * st.heads + 3) / 4));
    if (st.head_dim == 64)
        hipLaunchKernelGGL(attn_join_kernel<64>, grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(attn_join_kernel<128>, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

void plan_attn_tree(abq_attn_state *st, int most_parts)
{
    const int rows = st->max_q * (st->heads / st->kv_heads);
    // Blocks of 32 rows read a code once for two products, where there are two: 27 drafts of 4 heads per key head on 3 x 5500 tokens of
    // 4 bits 30.5 us, in blocks of 16 rows 32; 48 ragged contexts, 20 rows, 147.5 and 173.  (64 drafts on 4000 tokens, or 16 of 4 heads
    // on 4 x 2000, take the same in either: 20.8, 15.)  Up to 16 rows the second half would be empty, but the workgroups have half as many
    // threads, and twice as many of them fit a launch.
    const int64_t key_heads = (int64_t)st->seqs * st->kv_heads;
    st->block_rows = rows <= 16 && key_heads + 8 <= kMostThreads / (64 * tree_waves(1)) ? 16 : 32;
    const int64_t units = key_heads * ((rows + st->block_rows - 1) / st->block_rows);
    const int64_t steps = ((int64_t)st->max_k + kStep - 1) / kStep;
    // Eight waves of 16 rows, or two times four of 32, per compute unit, the more of a part's waves with a step or two the better: with
    // the cache's bytes from memory, and up to 16 rows, one sequence takes
    //   us in parts                        1     2     4     8    16    32
    //   1000 tokens, 32 key heads         11    10   9.3   8.2               (taken: 8)
    //   8000 tokens, 32                   46    29    20  17.7  18.4         (8)
    //   32768 tokens, 8                  168    90    50    29    20    19   (32)
    //   2 x 2000 tokens, 8                15    13    11     9    11         (8)
    //   4 x 4096 tokens, 32               33    31    32                     (2)
    // Up to three steps a wave the second launch costs as much as parts save, or more: one sequence of 8 key heads and one row, 500 tokens
    // in 1, 2 parts 7.3, 8.5 us, 700 tokens 8.6, 8.8; of 40 rows, 400 tokens in 1, 3 parts 10.5, 10.9, 500 in 1, 4 10.8, 9.8.
    const int waves = tree_waves(st->block_rows / 16);
    int64_t parts = steps > (waves == 8 ? 24 : 15) ? 2048 / waves / units : 1;
    const int64_t busy = steps / 4 < 8 || waves == 4 ? steps / 4 : steps / 8 > 8 ? steps / 8 : 8;
    parts = parts < busy ? parts : busy;
    // A wave has 32 steps at most, so that sequences much longer than the others are spread: 48 of up to 16384 tokens and 8 heads, 20
    // rows, in 1, 3, 5, 8 parts 230, 164, 153, 148 us, while 30 of 4000 and 32 heads, one row, take 175 in any number.
    const int64_t spread = (steps + 32 * waves - 1) / (32 * waves);
    parts = parts > spread ? parts : spread;
    parts = parts < most_parts ? parts : most_parts;
    // (launches within their limit: this one, rounded up, and the one that joins the parts, four rows of heads per workgroup)
    const int64_t row_blocks = (rows + st->block_rows - 1) / st->block_rows, most = kMostThreads / (64 * waves) / (units + 8 * row_blocks);
    parts = parts < most ? parts : most;
    if ((int64_t)st->seqs * st->max_q > 4 * kMostBlocks / st->heads)
        parts = 1;
    st->parts = parts < 1 ? 1 : (int)parts;
}

#define ABQ_TREE(B, A, D_, RT_) hipLaunchKernelGGL((attn_tree_kernel<B, A, D_, RT_>), grid, dim3(64 * tree_waves(RT_)), 0, stream, a)
#define ABQ_TREE_ROWS(B, A, D_)           \
    do {                                  \
        if (st.block_rows == 16)          \
            ABQ_TREE(B, A, D_, 1);        \
        else                              \
            ABQ_TREE(B, A, D_, 2);        \
    } while (0)
#define ABQ_TREE_DIM(B, A)                \
    do {                                  \
        if (st.head_dim == 64)            \
            ABQ_TREE_ROWS(B, A, 64);      \
        else                              \
            ABQ_TREE_ROWS(B, A, 128);     \
    } while (0)

hipError_t launch_attn_tree(const abq_attn_state &st, hipStream_t stream)
{
    TreeArgs a;
    a.c = st.cache;
    a.q = st.q;
    a.out = st.out;
    a.page_table = st.page_table;
    a.context = st.context;
    a.q_starts = st.q_starts;
    a.mask = st.mask;
    a.heads = st.heads;
    a.group = st.heads / st.kv_heads;
    a.seqs = st.seqs;
    a.max_q = st.max_q;
    a.max_pages = st.max_pages;
    a.row_blocks = (st.max_q * a.group + st.block_rows - 1) / st.block_rows;
    a.dtype = st.dtype;
    a.page_shift = __builtin_ctz((unsigned)st.cache.page_size);
    a.scale_log2 = st.scale * kLog2e;
    a.parts = attn_parts(st);
    const int64_t units = (int64_t)st.seqs * st.kv_heads * st.parts;
    const dim3 grid((unsigned)((units + 7) / 8 * 8 * a.row_blocks));
    if (st.cache.bits == 8) {
        if (st.cache.symmetric)
            ABQ_TREE_DIM(8, false);
        else
            ABQ_TREE_DIM(8, true);
    } else if (st.cache.symmetric)
        ABQ_TREE_DIM(4, false);
    else
        ABQ_TREE_DIM(4, true);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess || st.parts < 2 ? e : launch_attn_join(st, stream);
}

} // namespace abq
