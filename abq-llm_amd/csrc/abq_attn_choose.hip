// Which pages of a long context a query looks at: bounds of the keys of complete pages, and the choice by a bound of the scores.
// The formulas are those stated in abq_attention.h.
//
// A page's keys k of a channel lie between lo and hi, so q k <= max(q, 0) hi + min(q, 0) lo in that channel, and the sum over the channels is at
// least the score of any of its tokens (a published method: J. Tang et al., "Query-Aware Sparsity for Efficient Long-Context LLM Inference",
// ICML 2024).  With hi and lo beside each other that is one product of 2 head_dim numbers, in 8 bits on the
// matrix cores (16 x 16 x 64), exact in whole numbers: the choice is the same whatever the order of sums.
//
// Bounds are as many bytes as 2 tokens' keys, so reading them is little; what a choice takes is a chain: pages, bounds and query
// from memory 5 us (128 units of 512 pages, 17 MB), scores 1, the keys' range and one to four turns of the search for the threshold 0.6
// each, the list 0.9, and the launch.  One query for each of 16 x 8 heads and 512 pages 11.2 us, for 8 heads and 1500 pages 12.2 in two launches.
// Bounds are written at 4.4 TB/s where there are many (256 pages of 64 tokens and 32 heads, 69 MB, 15.8 us); sixteen sequences that all end a
// page take 4.2 us, a call that ends none 2.
#include "abq_decoding.h"
#include "abq_quant.h"

#include <type_traits>

namespace abq {

namespace {

__device__ __forceinline__ float max_of_wave(float x)
{
    x = max_across_quarters(x);
#pragma unroll
    for (int o = 1; o < 16; o *= 2)
        x = fmaxf(x, __shfl_xor(x, o));
    return x;
}

// ---------------------------------------------------------------------------------------------------------- bounds

struct BoundArgs {
    abq_kv_cache c;
    abq_kv_bounds b;
    const int32_t *slots;
    int64_t count;
    int page_shift, head_blocks, each; // each: slots that a workgroup looks through
};

// The elements of a lane's 16 bytes of codes, in order
template <int BITS> __device__ __forceinline__ float code_of(const uint32_t (&w)[4], int e)
{
    if (BITS == 8)
        return (float)(w[e / 4] >> (8 * (e & 3)) & 255);
    return (float)(w[e / 8] >> (4 * ((e & 1) * 4 + (e & 7) / 2)) & 15);
}

// Lanes that differ in bit O change parts: afterwards *keep has, in the lanes without the bit, both lanes' `first` (its own and *other's), in
// those with it both lanes' `second`
template <int O> __device__ __forceinline__ void exchange(float first, float second, int lane, float *keep, float *other)
{
    if constexpr (O >= 16) { // one operation: the upper halves of the one change places with the lower ones of the other
        const uint32_t f = __builtin_bit_cast(uint32_t, first), s = __builtin_bit_cast(uint32_t, second);
        uint32_t x, y;
        if constexpr (O == 32) {
            const auto r = __builtin_amdgcn_permlane32_swap(f, s, false, false);
            x = r[0], y = r[1];
        } else {
            const auto r = __builtin_amdgcn_permlane16_swap(f, s, false, false);
            x = r[0], y = r[1];
        }
        *keep = __builtin_bit_cast(float, x);
        *other = __builtin_bit_cast(float, y);
    } else {
        *keep = lane & O ? second : first;
        *other = __shfl_xor(lane & O ? first : second, O);
    }
}

// The largest of hi and the smallest of lo over the lanes that differ in the bits O, O / 2 .. LAST, a part of the N channels, from *c0 on, in each
template <int N, int O, int LAST> __device__ __forceinline__ void scatter(float *hi, float *lo, int lane, int *c0)
{
    if constexpr (O >= LAST) {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
            float keep, other;
            exchange<O>(hi[e], hi[N / 2 + e], lane, &keep, &other);
            hi[e] = fmaxf(keep, other);
            exchange<O>(lo[e], lo[N / 2 + e], lane, &keep, &other);
            lo[e] = fminf(keep, other);
        }
        *c0 += lane & O ? N / 2 : 0;
        scatter<N / 2, O / 2, LAST>(hi, lo, lane, c0);
    }
}

// A wave per head: it holds rows of R / 16 lanes, keeps the extrema of its own tokens in each lane, and joins them at the end.
template <int BITS, int D> __global__ __launch_bounds__(256) void kv_bound_kernel(BoundArgs a)
{
    constexpr int R = D * BITS / 8, kLanes = R / 16, kRows = 64 / kLanes, kEach = D / kLanes;
    const int lane = threadIdx.x & 63, li = lane % kLanes;
    // A prompt's pages end at every so many workgroups, which go round the eight XCDs: each eight of them in another order, lest all work be
    // one XCD's
    const uint32_t block = blockIdx.x ^ (blockIdx.x >> 3 & 7);
    const int head = block % a.head_blocks * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t i = (int64_t)(block / a.head_blocks) * a.each + lane;
    const int slot = lane < a.each && i < a.count ? a.slots[i] : -1;
    const int last = (1 << a.page_shift) - 1;
    uint64_t ends = __ballot(slot >= 0 && (slot & last) == last && (slot >> a.page_shift) < a.c.num_pages);
    if (head >= a.c.kv_heads)
        return;
    for (; ends; ends &= ends - 1) {
        const int page = __builtin_amdgcn_readlane(slot, __builtin_ctzll(ends)) >> a.page_shift;
        const int64_t row = ((int64_t)page * a.c.kv_heads + head) << a.page_shift;
        const uint8_t *codes = (const uint8_t *)a.c.k_codes + row * R;
        const float *scales = a.c.k_scales + (a.c.symmetric ? row : 2 * row);
        float hi[kEach], lo[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            hi[e] = -INFINITY;
            lo[e] = INFINITY;
        }
#pragma unroll 2
        for (int t0 = 0; t0 <= last; t0 += kRows) {
            const int t = min(t0 + lane / kLanes, last); // (a token twice is a token)
            const uint4 x = *(const uint4 *)(codes + t * R + 16 * li);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            const float scale = scales[t], zero = a.c.symmetric ? (float)(1 << (BITS - 1)) : scales[last + 1 + t];
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const float v = (code_of<BITS>(w, e) - zero) * scale;
                hi[e] = fmaxf(hi[e], v);
                lo[e] = fminf(lo[e], v);
            }
        }
        // Each exchange leaves a lane half of its channels, over twice the tokens: D / 64 of them in the end, over all (an exchange of all
        // channels each time took four times as long, and left the codes to a few lanes)
        int c0 = li * kEach;
        scatter<kEach, 32, kLanes>(hi, lo, lane, &c0);
        constexpr int kOwn = D / 64;
        float most = 0;
#pragma unroll
        for (int e = 0; e < kOwn; ++e)
            most = fmaxf(most, fmaxf(fabsf(hi[e]), fabsf(lo[e])));
        const QuantRow q = quant_row_params(max_of_wave(most), 0.f, 8, 1);
        const int64_t at = (int64_t)page * a.c.kv_heads + head;
        if (lane == 0)
            a.b.scales[at] = q.scale;
        int8_t *dst = a.b.codes + at * 2 * D + c0;
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
            dst[e] = (int8_t)quant_code_bits(hi[e], q);
            dst[D + e] = (int8_t)quant_code_bits(lo[e], q);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------- choice

struct ChooseArgs {
    abq_kv_cache c;
    abq_kv_bounds b;
    abq_rows q;
    const int32_t *page_table, *context, *q_starts;
    int32_t *blocks;
    int dtype, group, seqs, max_q, max_pages, first, last, count;
    int page_shift;
};

typedef __attribute__((ext_vector_type(4))) int int4v;

template <int CTRL> __device__ __forceinline__ float add_dpp(float x)
{
    return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// over the 16 lanes of a row: neighbours, pairs, mirrored halves, the other eight
__device__ __forceinline__ float sum_of_row(float x) { return add_dpp<0x128>(add_dpp<0x141>(add_dpp<0x4e>(add_dpp<0xb1>(x)))); }

template <int CTRL> __device__ __forceinline__ uint32_t most_dpp(uint32_t x)
{
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ uint32_t most_of_row(uint32_t x) { return most_dpp<0x128>(most_dpp<0x141>(most_dpp<0x4e>(most_dpp<0xb1>(x)))); }
// over a wave, as a scalar
__device__ __forceinline__ uint32_t most_of_wave(uint32_t x)
{
    x = most_of_row(x);
    const auto rows = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(rows[0], rows[1]);
    const auto halves = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __builtin_amdgcn_readfirstlane(max(halves[0], halves[1]));
}

// Floats as unsigned numbers of the same order, none of them 0, and back
__device__ __forceinline__ uint32_t ordered(float x)
{
    const uint32_t w = __builtin_bit_cast(uint32_t, x);
    return w & 0x80000000u ? ~w : w | 0x80000000u;
}
__device__ __forceinline__ float number_of(uint32_t key) { return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// What page p of n is chosen by
__device__ __forceinline__ uint32_t key_of(const ChooseArgs &a, int p, int n, bool in_cache, float score)
{
    return p < a.first || p >= n - a.last ? ~0u : in_cache ? ordered(score) : 0;
}

// What a wave asks for at once: bounds of COUNT tiles of 16 pages, as columns of the product, those of tile i from page p0 + i * step on.
// Page numbers are asked for before the number of pages is known, their bounds before the query is: three loads one behind the
// other instead of five.
template <int D, int COUNT> struct Tiles {
    static constexpr int kCount = COUNT, kChunks = D / 64;
    int page[kCount];
    int4v bounds[kCount][2][kChunks];
    float scale[kCount];

    __device__ __forceinline__ void ask_pages(const ChooseArgs &a, const int32_t *pages, int p0, int step)
    {
#pragma unroll
        for (int i = 0; i < kCount; ++i)
            page[i] = pages[min(p0 + step * i + (int)(threadIdx.x & 15), a.max_pages - 1)];
    }
    __device__ __forceinline__ void ask_bounds(const ChooseArgs &a, int head, int p0, int step, int n)
    {
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            if (p0 + step * i >= n)
                continue;
            const int64_t at = (int64_t)(in_cache(a, i) ? page[i] : 0) * a.c.kv_heads + head;
            const int8_t *bound = a.b.codes + at * 2 * D + 16 * (threadIdx.x >> 4 & 3);
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                bounds[i][0][j] = *(const int4v *)(bound + 64 * j);
                bounds[i][1][j] = *(const int4v *)(bound + D + 64 * j);
            }
            scale[i] = a.b.scales[at];
        }
    }
    __device__ __forceinline__ bool in_cache(const ChooseArgs &a, int i) const { return (uint32_t)page[i] < (uint32_t)a.c.num_pages; }
};

// Rows of queries as the product takes sixteen of them, in LDS: what is positive of their codes, what is negative (padded against bank conflicts),
// and their scales.  A wave quantises a row: what every wave would do for itself otherwise is most of the kernel's time.
template <int D, int ROWS = 16> struct Rows {
    __align__(16) int8_t codes[2][ROWS][D + 16];
    float scales[ROWS];

    // rows[i] goes to row i0 + i * step; NULL: it stays as it is
    template <int N> __device__ __forceinline__ void quantise(const uint16_t *const (&rows)[N], int i0, int step, int dtype)
    {
        constexpr int kEach = D / 64;
        const int lane = threadIdx.x & 63;
        uint32_t w[N];
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (rows[i])
                w[i] = kEach == 2 ? ((const uint32_t *)rows[i])[lane] : rows[i][lane];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (!rows[i])
                continue;
            float x[2];
            x[0] = dtype == ABQ_BF16 ? value16<ABQ_BF16>(w[i]) : value16<ABQ_F16>(w[i]);
            x[1] = kEach == 1 ? 0 : dtype == ABQ_BF16 ? value16<ABQ_BF16>(w[i] >> 16) : value16<ABQ_F16>(w[i] >> 16);
            const QuantRow q = quant_row_params(max_of_wave(fmaxf(fabsf(x[0]), fabsf(x[1]))), 0.f, 8, 1);
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int c = (int8_t)quant_code_bits(x[e], q);
                codes[0][i0 + i * step][kEach * lane + e] = (int8_t)max(c, 0);
                codes[1][i0 + i * step][kEach * lane + e] = (int8_t)min(c, 0);
            }
            if (lane == 0)
                scales[i0 + i * step] = q.scale;
        }
    }
    // Of sixteen from row r on, lane (t, g): the channels 64 j + 16 g .. + 15 of row t, and the scales of rows 4 g .. 4 g + 3, whose sums it gets
    __device__ __forceinline__ void read(int r, int4v (&up)[D / 64], int4v (&down)[D / 64], float (&scale)[4]) const
    {
        const int t = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            up[j] = *(const int4v *)&codes[0][r + t][64 * j + 16 * g];
            down[j] = *(const int4v *)&codes[1][r + t][64 * j + 16 * g];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            scale[i] = scales[r + 4 * g + i];
    }
};

// Sums of a tile's pages: lane (t, g) has page t's of rows 4 g .. 4 g + 3
template <int D, int COUNT> __device__ __forceinline__ int4v sums_of(const Tiles<D, COUNT> &tiles, int i, const int4v (&up)[D / 64], const int4v (&down)[D / 64])
{
    int4v acc = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(up[j], tiles.bounds[i][0][j], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(down[j], tiles.bounds[i][1][j], acc, 0, 0, 0);
    }
    return acc;
}

// A query row of a sequence and a key head
struct ChooseUnit {
    int seq, draft, head;
};
__device__ __forceinline__ ChooseUnit choose_unit(const ChooseArgs &a, uint32_t unit)
{
    return {(int)(unit / a.c.kv_heads / a.max_q), (int)(unit / a.c.kv_heads % a.max_q), (int)(unit % a.c.kv_heads)};
}
__device__ __forceinline__ int complete_pages(const ChooseArgs &a, int seq) { return min(max(a.context[seq], 0) >> a.page_shift, a.max_pages); }

// Scores of all pages of a query row into LDS, by a workgroup
template <int D, int WAVES> __device__ __forceinline__ void score_pages(const ChooseArgs &a, const ChooseUnit &u, uint32_t *keys)
{
    __shared__ Rows<D> rows;
    using T = Tiles<D, 4>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = lane & 15, g = lane >> 4;
    const int32_t *pages = a.page_table + (int64_t)u.seq * a.max_pages;
    constexpr int kStep = 16 * WAVES, kRound = kStep * T::kCount;
    T tiles;
    tiles.ask_pages(a, pages, 16 * wave, kStep);
    const SeqRows own = seq_rows(a.q_starts, u.seq, a.q.rows);
    const int n = complete_pages(a, u.seq);
    if (u.draft >= own.count || n <= a.count)
        return;
    tiles.ask_bounds(a, u.head, 16 * wave, kStep, n);
    for (int h0 = 0; h0 < a.group; h0 += 16) {
        if (h0 > 0)
            __syncthreads();
        for (int h = wave; h < min(a.group - h0, 16); h += WAVES) {
            const uint16_t *row[1] = {(const uint16_t *)a.q.data + (own.first + u.draft) * a.q.row_stride + (int64_t)(u.head * a.group + h0 + h) * a.q.head_stride};
            rows.quantise(row, h, 0, a.dtype);
        }
        __syncthreads();
        int4v up[D / 64], down[D / 64];
        float scale[4];
        rows.read(0, up, down, scale);
        for (int p0 = 16 * wave; p0 < n; p0 += kRound) {
            if (p0 >= kRound || h0 > 0) { // (else they are there)
                tiles.ask_pages(a, pages, p0, kStep);
                tiles.ask_bounds(a, u.head, p0, kStep, n);
            }
#pragma unroll
            for (int i = 0; i < T::kCount; ++i) {
                const int p = p0 + kStep * i + t;
                if (p - t >= n)
                    continue;
                const int4v acc = sums_of(tiles, i, up, down);
                float score = -INFINITY; // (rows behind the last head are whatever is there: their sums are not looked at)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    score = h0 + 4 * g + k < a.group ? fmaxf(score, (float)acc[k] * scale[k]) : score;
                score = max_across_quarters(score);
                if (g == 0 && p < n) {
                    if (h0 > 0)
                        score = fmaxf(score, __builtin_bit_cast(float, keys[p]));
                    if (h0 + 16 < a.group)
                        keys[p] = __builtin_bit_cast(uint32_t, score);
                    else
                        keys[p] = key_of(a, p, n, tiles.in_cache(a, i), score * tiles.scale[i]);
                }
            }
        }
    }
}

// The numbers of the `want` largest of n > want keys in LDS, lower numbers first among equal keys, in order, by a workgroup
template <int WAVES> __device__ __forceinline__ void write_largest(const uint32_t *keys, int n, int want, int32_t *out)
{
    __shared__ uint32_t in_wave[2][8][16];
    __shared__ uint2 ends[4][16];
    constexpr int kThreads = 64 * WAVES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = lane & 15, g = lane >> 4;
    const int rounded = (n + kThreads - 1) / kThreads * kThreads;
    const uint32_t first = threadIdx.x < n ? keys[threadIdx.x] : 0, second = threadIdx.x + kThreads < n ? keys[threadIdx.x + kThreads] : 0;
    // The least key and the largest of pages that are not chosen anyway: the former is among what `want` reach, and so much of the keys' bits is
    // the same in all: 125 pages of scores between 100 and 300 take 6.9 us, 8.4 from the keys' first bit on.  (Complements, and sums that wrap around, make both a largest one, and nothing of a key that is passed over.)
    uint32_t from = 0, to = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint32_t key = i < kThreads ? first : i < 2 * kThreads ? second : keys[i];
        from = max(from, ~key);
        to = max(to, key + 1);
    }
    from = most_of_row(from);
    to = most_of_row(to);
    if (t == 0)
        ends[g][wave] = uint2{from, to};
    __syncthreads();
    const uint2 end = t < WAVES ? ends[g][t] : uint2{0, 0};
    from = ~most_of_wave(end.x);
    to = most_of_wave(end.y) - 1;
    // The largest number that at least `want` keys reach, three bits at a time; `exact`: reached by no more than those.  Each wave counts its
    // own keys; then lane (w, j) of every wave has wave w's count of those that reach the j-th of seven numbers, so that a turn is one
    // write, one barrier and one read, and what follows from it is the same in all waves.
    uint32_t least = from;
    bool exact = false;
    for (int bits = to > from ? 32 - __builtin_clz(to - from) : 0, round = 0; bits > 0 && !exact; bits -= 3, ++round) {
        const int shift = max(bits - 3, 0);
        uint32_t count[7] = {};
        auto tally = [&](uint32_t key) {
            const uint32_t digit = key >= least ? (key - least) >> shift : 0;
#pragma unroll
            for (int j = 0; j < 7; ++j)
                count[j] += __popcll(__ballot(digit > (uint32_t)j));
        };
        tally(first);
        tally(second);
        for (int i = threadIdx.x + 2 * kThreads; i < rounded; i += kThreads)
            tally(i < n ? keys[i] : 0);
        uint32_t mine = count[0];
#pragma unroll
        for (int j = 1; j < 7; ++j)
            mine = lane == j ? count[j] : mine;
        if (lane < 7)
            in_wave[round & 1][lane][wave] = mine;
        __syncthreads();
        // (whole numbers below 2^16; counts do not grow with j)
        const uint32_t low = in_wave[round & 1][g][t], high = in_wave[round & 1][4 + g][t];
        const float total_low = sum_of_row(t < WAVES ? (float)low : 0.f), total_high = sum_of_row(t < WAVES && g < 3 ? (float)high : 0.f);
        constexpr uint64_t kRows = 0x0001000100010001ull;
        const int digit = __popcll(__ballot(total_low >= (float)want) & kRows) + __popcll(__ballot(total_high >= (float)want) & kRows);
        const uint64_t just_low = __ballot(total_low == (float)want), just_high = __ballot(total_high == (float)want);
        least += (uint32_t)digit << shift;
        exact = digit > 0 && ((digit > 4 ? just_high : just_low) >> (16 * ((digit - 1) & 3)) & 1);
    }
    // How many of those that are just as large there is room for: all, or what the larger ones leave
    int room = want;
    if (!exact) {
        __syncthreads();
        int larger = 0;
        for (int i = threadIdx.x; i < rounded; i += kThreads)
            larger += __popcll(__ballot(i < n && keys[i] > least));
        if (lane == 0)
            in_wave[0][0][wave] = larger;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
            room -= in_wave[0][0][w];
    }
    // in order: larger ones and equal ones before each page, in the two halves of a word (n < 2^16)
    uint32_t before = 0;
    for (int base = 0, round = 0; base < n; base += kThreads, ++round) {
        const int i = base + threadIdx.x;
        const uint32_t key = i < n ? keys[i] : 0;
        const bool larger = i < n && key > least, equal = i < n && key == least;
        const uint64_t l = __ballot(larger), e = __ballot(equal), below = (1ull << lane) - 1;
        uint32_t mine = __popcll(l & below) | __popcll(e & below) << 16;
        if (lane == 0)
            in_wave[round & 1][7][wave] = __popcll(l) | __popcll(e) << 16;
        __syncthreads();
        uint32_t all = before;
        mine += before;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const uint32_t x = in_wave[round & 1][7][w];
            mine += w < wave ? x : 0;
            all += x;
        }
        before = all;
        const int equal_before = mine >> 16, at = (mine & 0xffff) + min(equal_before, room);
        if (larger || (equal && equal_before < room))
            out[at] = i;
    }
}

// A workgroup per query and key head: scores of all its pages into LDS, or from `scored` ([unit][max_pages]), and the choice among them.
template <int D, int WAVES, bool SCORED> __global__ __launch_bounds__(64 * WAVES) void attn_choose_kernel(ChooseArgs a, const uint32_t *scored)
{
    extern __shared__ uint32_t keys[]; // [max_pages]
    constexpr int kThreads = 64 * WAVES;
    const ChooseUnit u = choose_unit(a, blockIdx.x);
    if constexpr (!SCORED)
        score_pages<D, WAVES>(a, u, keys);
    const SeqRows own = seq_rows(a.q_starts, u.seq, a.q.rows);
    if (u.draft >= own.count)
        return;
    const int n = complete_pages(a, u.seq), want = a.count;
    int32_t *out = a.blocks + ((int64_t)(own.first + u.draft) * a.c.kv_heads + u.head) * want;
    if (n <= want) {
        for (int i = threadIdx.x; i < want; i += kThreads)
            out[i] = i < n ? i : -1;
        return;
    }
    if constexpr (SCORED)
        for (int i = threadIdx.x; i < n; i += kThreads)
            keys[i] = scored[(int64_t)blockIdx.x * a.max_pages + i];
    __syncthreads();
    write_largest<WAVES>(keys, n, want, out);
}

// The scores alone, a workgroup for kScorePages pages of a sequence and key head and for some of the sequence's drafts, whose rows it goes over
// with the bounds in registers.  Rows of all its drafts' heads fill the product's sixteen; each goes into its draft's largest.
constexpr int kScoreWaves = 4, kScoreTiles = 2, kScorePages = 16 * kScoreWaves * kScoreTiles;
// 32 rows of queries a workgroup, quantised at once (7 x 5 drafts of 4 heads, 1250 pages 20.7 us, sixteen and sixteen 21.7; 16 x 5 28.4 and 32.3):
// more of them in turn take longer than reading the bounds again
constexpr int kScoreRows = 32;
constexpr int score_drafts(int group) { return group >= kScoreRows ? 1 : kScoreRows / group; }

template <int D> __global__ __launch_bounds__(64 * kScoreWaves) void attn_score_kernel(ChooseArgs a, uint32_t *scored)
{
    __shared__ Rows<D, kScoreRows> rows;
    __shared__ uint32_t keys[score_drafts(1)][kScorePages];
    __shared__ float scales[kScorePages]; // of bounds; -inf: the page is not in the cache
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = lane & 15, g = lane >> 4;
    const int each = score_drafts(a.group);
    const uint32_t parts = (a.max_pages + kScorePages - 1) / kScorePages, turns = (a.max_q + each - 1) / each, unit = blockIdx.x / parts / turns;
    const int begin = (int)(blockIdx.x % parts) * kScorePages, d0 = (int)(blockIdx.x / parts % turns) * each, seq = unit / a.c.kv_heads, head = unit % a.c.kv_heads;
    constexpr int kStep = 16 * kScoreWaves;
    Tiles<D, kScoreTiles> tiles;
    tiles.ask_pages(a, a.page_table + (int64_t)seq * a.max_pages, begin + 16 * wave, kStep);
    const SeqRows own = seq_rows(a.q_starts, seq, a.q.rows);
    const int all = complete_pages(a, seq), n = min(all - begin, kScorePages), some = min(min(own.count, a.max_q) - d0, each);
    if (some <= 0 || all <= a.count || n <= 0)
        return;
    tiles.ask_bounds(a, head, begin + 16 * wave, kStep, all);
    uint32_t *out = scored + (((int64_t)seq * a.max_q + d0) * a.c.kv_heads + head) * a.max_pages + begin; // of draft d0
    const int count = some * a.group;
    const bool one = some == 1 && count <= 16; // (no other row has a part in a page's score)
    if (!one)
        for (int i = threadIdx.x; i < some * kScorePages; i += 64 * kScoreWaves)
            (&keys[0][0])[i] = 0;
    for (int r0 = 0; r0 < count; r0 += 16) {
        if (r0 % kScoreRows == 0) {
            if (r0 > 0)
                __syncthreads();
            auto quantise = [&](auto n) { // (half as many loads and branches where there are no more rows: 8 x 8000 pages 25 us, 27 without)
                const uint16_t *row[decltype(n)::value];
#pragma unroll
                for (int i = 0; i < decltype(n)::value; ++i) {
                    const int r = r0 + kScoreWaves * i + wave;
                    row[i] = r < count ? (const uint16_t *)a.q.data + (own.first + d0 + r / a.group) * a.q.row_stride + (int64_t)(head * a.group + r % a.group) * a.q.head_stride : nullptr;
                }
                rows.quantise(row, wave, kScoreWaves, a.dtype);
            };
            if (count - r0 <= 16)
                quantise(std::integral_constant<int, 16 / kScoreWaves>());
            else
                quantise(std::integral_constant<int, kScoreRows / kScoreWaves>());
            __syncthreads();
        }
        int4v up[D / 64], down[D / 64];
        float scale[4];
        rows.read(r0 % kScoreRows, up, down, scale);
        int draft[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            draft[k] = r0 + 4 * g + k < count ? (r0 + 4 * g + k) / a.group : -1;
#pragma unroll
        for (int i = 0; i < kScoreTiles; ++i) {
            const int p = kStep * i + 16 * wave + t;
            if (p - t >= n)
                continue;
            const int4v acc = sums_of(tiles, i, up, down);
            if (one) {
                float score = -INFINITY;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    score = draft[k] == 0 ? fmaxf(score, (float)acc[k] * scale[k]) : score;
                score = max_across_quarters(score);
                if (g == 0 && p < n)
                    out[p] = key_of(a, begin + p, all, tiles.in_cache(a, i), score * tiles.scale[i]);
                continue;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (draft[k] >= 0)
                    atomicMax(&keys[draft[k]][p], ordered((float)acc[k] * scale[k]));
            if (g == 0)
                scales[p] = tiles.in_cache(a, i) ? tiles.scale[i] : -INFINITY;
        }
    }
    if (one)
        return;
    __syncthreads();
    for (int i = threadIdx.x; i < some * kScorePages; i += 64 * kScoreWaves) {
        const int d = i / kScorePages, p = i % kScorePages;
        if (p < n)
            out[(int64_t)d * a.c.kv_heads * a.max_pages + p] = key_of(a, begin + p, all, scales[p] != -INFINITY, number_of(keys[d][p]) * scales[p]);
    }
}

} // namespace

#define ABQ_BOUND(B)                                                                                       \
    do {                                                                                                   \
        if (c.head_dim == 64)                                                                              \
            hipLaunchKernelGGL((kv_bound_kernel<B, 64>), grid, dim3(256), 0, stream, a);                   \
        else                                                                                               \
            hipLaunchKernelGGL((kv_bound_kernel<B, 128>), grid, dim3(256), 0, stream, a);                  \
    } while (0)

// Few slots may be of as many sequences, whose pages may all end at once; many are a prompt's, one of so many ends a page, and workgroups
// that find none are not for nothing (16384 slots, 256 pages of 32 heads: 42 us with 8 slots a workgroup, whose least is the launch of 16384)
int bound_slots(const abq_kv_cache &c, int64_t count) { return count <= 1024 ? 1 : c.page_size < 64 ? c.page_size : 64; }

hipError_t launch_kv_bound(const abq_kv_cache &c, const abq_kv_bounds &bounds, const int32_t *slots, int64_t count, hipStream_t stream)
{
    if (count == 0)
        return hipSuccess;
    BoundArgs a = {c, bounds, slots, count, __builtin_ctz((unsigned)c.page_size), (c.kv_heads + 3) / 4, bound_slots(c, count)};
    const dim3 grid((unsigned)(((count + a.each - 1) / a.each * a.head_blocks + 7) / 8 * 8));
    if (c.bits == 8)
        ABQ_BOUND(8);
    else
        ABQ_BOUND(4);
    return hipGetLastError();
}

template <int D, int WAVES, bool SCORED> static hipError_t choose(const ChooseArgs &a, const uint32_t *scored, int64_t units, hipStream_t stream)
{
    const size_t lds = sizeof(uint32_t) * a.max_pages;
    // A launch gets 64 KB unasked, of which the kernel's own arrays may take 7.  The limit is the process's: the same one each time, so that
    // no call lowers it between another thread's asking and its launch.
    if (lds > 48 << 10) {
        const hipError_t e = hipFuncSetAttribute((const void *)attn_choose_kernel<D, WAVES, SCORED>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)sizeof(uint32_t) * kMostChosen);
        if (e != hipSuccess)
            return e;
    }
    hipLaunchKernelGGL((attn_choose_kernel<D, WAVES, SCORED>), dim3((unsigned)units), dim3(64 * WAVES), lds, stream, a, scored);
    return hipGetLastError();
}

template <int D> static hipError_t choose(const ChooseArgs &a, int64_t units, int likely, uint32_t *scored, hipStream_t stream)
{
    if (scored) {
        const int64_t parts = (a.max_pages + kScorePages - 1) / kScorePages, turns = (a.max_q + score_drafts(a.group) - 1) / score_drafts(a.group);
        hipLaunchKernelGGL(attn_score_kernel<D>, dim3((unsigned)(a.seqs * a.c.kv_heads * parts * turns)), dim3(64 * kScoreWaves), 0, stream, a, scored);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess)
            return e;
        return likely <= 1024 || units > 64 ? choose<D, 8, true>(a, scored, units, stream) : choose<D, 16, true>(a, scored, units, stream);
    }
    // Waves: enough to score all pages in a round of 64 a wave, but no more than leave two (eight waves) or four workgroups to a compute unit
    // where there are more of these than units.  128 channels, us with 4, 8, 16 waves: 32 of 125 pages 6.9, 7.0, 8.1; 128 of 512 12.3, 11.2, 12.3;
    // 256 of 1200 27, 23.4, 22.7; 280 of 1250 32, 28, 35; 512 of 1200 43, 38, 45; 2048 of 1000 81, 88, 128
    if (likely <= 256 || units > 512)
        return choose<D, 4, false>(a, nullptr, units, stream);
    return likely <= 512 || units > 256 ? choose<D, 8, false>(a, nullptr, units, stream) : choose<D, 16, false>(a, nullptr, units, stream);
}

// A launch of their own for the scores: where few workgroups would each have many pages, and where several drafts share a sequence's bounds.
// us in one launch and in two, one draft: 8 units of 600 pages 11.9 and 10.5, of 1500 20.5 and 12.2, of 8000 80 and 25; 64 of 1500 21 and 16;
// but 8 of 300 8.5 and 10, 128 of 1200 19.9 either way.  Drafts: 7 x 5 of 8 heads, 600 pages 17.9 and 16.5, 1250 28.7 and 20.7; 64 of 32
// heads, 600 pages 52 and 31.7; but 2 x 27 of 8 heads, 600 pages 18.5 and 18.9.
size_t choose_workspace_bytes(int seqs, int max_q, int kv_heads, int max_pages, int likely)
{
    const double units = (double)seqs * max_q * kv_heads, blocks = units * ((max_pages + kScorePages - 1) / kScorePages);
    const bool two = likely > 512 && (units <= 64 || max_q > 1) && blocks <= kMostBlocks;
    return two ? (size_t)seqs * max_q * kv_heads * max_pages * sizeof(uint32_t) : 0;
}

hipError_t launch_attn_choose(const ChooseCall &call, hipStream_t stream)
{
    if (call.q.rows == 0)
        return hipSuccess;
    const ChooseArgs a = {call.cache, call.bounds, call.q, call.page_table, call.context, call.q_starts, call.blocks, call.dtype, call.heads / call.cache.kv_heads,
                          call.seqs, call.max_q, call.max_pages, call.first, call.last, call.count, __builtin_ctz((unsigned)call.cache.page_size)};
    const int64_t units = (int64_t)call.seqs * call.max_q * call.cache.kv_heads;
    const size_t need = choose_workspace_bytes(call.seqs, call.max_q, call.cache.kv_heads, call.max_pages, call.likely);
    uint32_t *scored = need && call.workspace_bytes >= need ? (uint32_t *)call.workspace : nullptr;
    return call.cache.head_dim == 64 ? choose<64>(a, units, call.likely, scored, stream) : choose<128>(a, units, call.likely, scored, stream);
}

} // namespace abq
