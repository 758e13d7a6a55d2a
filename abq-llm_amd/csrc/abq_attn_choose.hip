// Which pages of a long context a query looks at: bounds of the keys of complete pages, and the choice by a bound of the scores.
// The formulas are those stated in abq_attention.h.
//
// A page's keys k of a channel lie between lo and hi, so q k <= max(q, 0) hi + min(q, 0) lo in that channel, and the sum over the channels is at
// least the score of any of its tokens.  With hi and lo beside each other that is one product of 2 head_dim numbers, in 8 bits on the
// matrix cores (16 x 16 x 64), exact in whole numbers: the choice is the same whatever the order of sums.
#include "abq_decoding.h"
#include "abq_quant.h"

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
    int page_shift, head_blocks;
};

constexpr int kBoundSlots = 8; // that a workgroup looks through

// The elements of a lane's 16 bytes of codes, in order
template <int BITS> __device__ __forceinline__ float code_of(const uint32_t (&w)[4], int e)
{
    if (BITS == 8)
        return (float)(w[e / 4] >> (8 * (e & 3)) & 255);
    return (float)(w[e / 8] >> (4 * ((e & 1) * 4 + (e & 7) / 2)) & 15);
}

// The largest of hi and the smallest of lo over the lanes that differ in the bits O, O / 2 .. LAST, a part of the N channels, from *c0 on, in each
template <int N, int O, int LAST> __device__ __forceinline__ void scatter(float *hi, float *lo, int lane, int *c0)
{
    if constexpr (O >= LAST) {
        const bool upper = lane & O;
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
            const float h = __shfl_xor(upper ? hi[e] : hi[N / 2 + e], O), l = __shfl_xor(upper ? lo[e] : lo[N / 2 + e], O);
            hi[e] = fmaxf(upper ? hi[N / 2 + e] : hi[e], h);
            lo[e] = fminf(upper ? lo[N / 2 + e] : lo[e], l);
        }
        *c0 += upper ? N / 2 : 0;
        scatter<N / 2, O / 2, LAST>(hi, lo, lane, c0);
    }
}

// A wave per head: it holds rows of R / 16 lanes, keeps the extrema of its own tokens in each lane, and joins them at the end.
template <int BITS, int D> __global__ __launch_bounds__(256) void kv_bound_kernel(BoundArgs a)
{
    constexpr int R = D * BITS / 8, kLanes = R / 16, kRows = 64 / kLanes, kEach = D / kLanes;
    const int lane = threadIdx.x & 63, li = lane % kLanes;
    const int head = blockIdx.x % a.head_blocks * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t i = (int64_t)(blockIdx.x / a.head_blocks) * kBoundSlots + lane;
    const int slot = lane < kBoundSlots && i < a.count ? a.slots[i] : -1;
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
            const uint4 x = *(const uint4 *)(codes + (int64_t)t * R + 16 * li);
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

// Floats as unsigned numbers of the same order
__device__ __forceinline__ uint32_t ordered(float x)
{
    const uint32_t w = __builtin_bit_cast(uint32_t, x);
    return w & 0x80000000u ? ~w : w | 0x80000000u;
}

// What a wave asks for at once: bounds of four tiles of 16 pages, as columns of the product
template <int D> struct Tiles {
    static constexpr int kCount = 4, kChunks = D / 64;
    int page[kCount];
    int4v bounds[kCount][2][kChunks];
    float scale[kCount];
};

// A query row of a sequence and a key head
struct ChooseUnit {
    int seq, draft, head;
};
__device__ __forceinline__ ChooseUnit choose_unit(const ChooseArgs &a, uint32_t unit)
{
    return {(int)(unit / a.c.kv_heads / a.max_q), (int)(unit / a.c.kv_heads % a.max_q), (int)(unit % a.c.kv_heads)};
}
__device__ __forceinline__ int complete_pages(const ChooseArgs &a, int seq) { return min(max(a.context[seq], 0) >> a.page_shift, a.max_pages); }

// Scores of the pages from begin on, as many as there are before end, by all waves of a workgroup: keys[p - begin] for page p
template <int D, int WAVES> __device__ __forceinline__ void score_pages(const ChooseArgs &a, const ChooseUnit &u, int begin, int end, uint32_t *keys)
{
    __shared__ __align__(16) int8_t rows[2][16][D + 16]; // of queries: what is positive of them, what is negative (padded against bank conflicts)
    __shared__ float row_scales[16];
    constexpr int kChunks = D / 64;
    using T = Tiles<D>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = lane & 15, g = lane >> 4;
    const int32_t *pages = a.page_table + (int64_t)u.seq * a.max_pages;
    T tiles;
    // Page numbers are asked for before the number of pages is known, their bounds before the query is: three loads one behind the other
    // instead of five
    auto ask_pages = [&](int p0) {
#pragma unroll
        for (int i = 0; i < T::kCount; ++i)
            tiles.page[i] = pages[min(p0 + 16 * WAVES * i + t, a.max_pages - 1)];
    };
    auto ask_bounds = [&](int p0, int n) {
#pragma unroll
        for (int i = 0; i < T::kCount; ++i) {
            if (p0 + 16 * WAVES * i >= n)
                continue;
            const int64_t at = (int64_t)((uint32_t)tiles.page[i] < (uint32_t)a.c.num_pages ? tiles.page[i] : 0) * a.c.kv_heads + u.head;
            const int8_t *bound = a.b.codes + at * 2 * D + 16 * g;
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                tiles.bounds[i][0][j] = *(const int4v *)(bound + 64 * j);
                tiles.bounds[i][1][j] = *(const int4v *)(bound + D + 64 * j);
            }
            tiles.scale[i] = a.b.scales[at];
        }
    };
    ask_pages(begin + 16 * wave);
    const SeqRows own = seq_rows(a.q_starts, u.seq, a.q.rows);
    const int all = complete_pages(a, u.seq), n = min(all, end);
    if (u.draft >= own.count || all <= a.count || begin >= n)
        return;
    ask_bounds(begin + 16 * wave, n);
    const int64_t q_row = own.first + u.draft;

    for (int h0 = 0; h0 < a.group; h0 += 16) {
        // Heads h0 .. h0 + 15 as rows of the product, a wave quantising each: what every wave would do for itself otherwise is most of the
        // kernel's time.  (Rows behind the last head are whatever is there: their sums are not looked at.)
        if (h0 > 0)
            __syncthreads();
        for (int h = wave; h < min(a.group - h0, 16); h += WAVES) {
            constexpr int kEach = D / 64;
            const uint16_t *src = (const uint16_t *)a.q.data + q_row * a.q.row_stride + (int64_t)(u.head * a.group + h0 + h) * a.q.head_stride + kEach * lane;
            float x[kEach], most = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                x[i] = a.dtype == ABQ_BF16 ? value16<ABQ_BF16>(src[i]) : value16<ABQ_F16>(src[i]);
                most = fmaxf(most, fabsf(x[i]));
            }
            const QuantRow row = quant_row_params(max_of_wave(most), 0.f, 8, 1);
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int c = (int8_t)quant_code_bits(x[i], row);
                rows[0][h][kEach * lane + i] = (int8_t)max(c, 0);
                rows[1][h][kEach * lane + i] = (int8_t)min(c, 0);
            }
            if (lane == 0)
                row_scales[h] = row.scale;
        }
        __syncthreads();
        // lane (t, g): the channels 64 j + 16 g .. + 15 of head h0 + t, and the scales of heads h0 + 4 g .. + 3, whose sums it gets
        int4v up[kChunks], down[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            up[j] = *(const int4v *)&rows[0][t][64 * j + 16 * g];
            down[j] = *(const int4v *)&rows[1][t][64 * j + 16 * g];
        }
        float scale[4];
        bool heads[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            scale[i] = row_scales[4 * g + i];
            heads[i] = h0 + 4 * g + i < a.group;
        }
        constexpr int kRound = 16 * WAVES * T::kCount;
        for (int p0 = begin + 16 * wave; p0 < n; p0 += kRound) {
            if (p0 >= begin + kRound || h0 > 0) { // (else they are there)
                ask_pages(p0);
                ask_bounds(p0, n);
            }
#pragma unroll
            for (int i = 0; i < T::kCount; ++i) {
                const int p = p0 + 16 * WAVES * i + t;
                if (p - t >= n)
                    continue;
                int4v acc = {0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < kChunks; ++j) {
                    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(up[j], tiles.bounds[i][0][j], acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(down[j], tiles.bounds[i][1][j], acc, 0, 0, 0);
                }
                // (lane (t, g) has page t's sums of heads 4 g .. 4 g + 3)
                float score = -INFINITY;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    score = heads[k] ? fmaxf(score, (float)acc[k] * scale[k]) : score;
                score = max_across_quarters(score);
                if (g == 0 && p < n) {
                    const bool in_cache = (uint32_t)tiles.page[i] < (uint32_t)a.c.num_pages;
                    if (h0 > 0)
                        score = fmaxf(score, __builtin_bit_cast(float, keys[p - begin]));
                    if (h0 + 16 < a.group)
                        keys[p - begin] = __builtin_bit_cast(uint32_t, score);
                    else
                        keys[p - begin] = p < a.first || p >= all - a.last ? ~0u : in_cache ? ordered(score * tiles.scale[i]) : 0;
                }
            }
        }
    }
}

// The numbers of the `want` largest of n > want keys in LDS, lower numbers first among equal keys, in order, by a workgroup
template <int WAVES> __device__ __forceinline__ void write_largest(const uint32_t *keys, int n, int want, int32_t *out)
{
    __shared__ uint32_t in_wave[2][8][16];
    constexpr int kThreads = 64 * WAVES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = lane & 15, g = lane >> 4;
    // The largest number that at least `want` keys reach, three bits at a time; `exact`: reached by no more than those.  Each wave counts its
    // own keys; then lane (w, j) of every wave has wave w's count of those that reach the j-th of seven numbers, so that a turn is one
    // write, one barrier and one read, and what follows from it is the same in all waves.
    uint32_t least = 0;
    bool exact = false;
    const int rounded = (n + kThreads - 1) / kThreads * kThreads;
    const uint32_t first = threadIdx.x < n ? keys[threadIdx.x] : 0, second = threadIdx.x + kThreads < n ? keys[threadIdx.x + kThreads] : 0;
    for (int shift = 30, round = 0; shift >= 0 && !exact; shift -= 3, ++round) {
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
        score_pages<D, WAVES>(a, u, 0, a.max_pages, keys);
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

// The scores alone, a workgroup for each kScorePages of them
constexpr int kScoreWaves = 4, kScorePages = 16 * kScoreWaves * 2;

template <int D> __global__ __launch_bounds__(64 * kScoreWaves) void attn_score_kernel(ChooseArgs a, uint32_t *scored)
{
    const uint32_t parts = (a.max_pages + kScorePages - 1) / kScorePages, unit = blockIdx.x / parts;
    const int begin = (int)(blockIdx.x % parts) * kScorePages;
    score_pages<D, kScoreWaves>(a, choose_unit(a, unit), begin, begin + kScorePages, scored + (int64_t)unit * a.max_pages + begin);
}

} // namespace

#define ABQ_BOUND(B)                                                                                       \
    do {                                                                                                   \
        if (c.head_dim == 64)                                                                              \
            hipLaunchKernelGGL((kv_bound_kernel<B, 64>), grid, dim3(256), 0, stream, a);                   \
        else                                                                                               \
            hipLaunchKernelGGL((kv_bound_kernel<B, 128>), grid, dim3(256), 0, stream, a);                  \
    } while (0)

hipError_t launch_kv_bound(const abq_kv_cache &c, const abq_kv_bounds &bounds, const int32_t *slots, int64_t count, hipStream_t stream)
{
    if (count == 0)
        return hipSuccess;
    BoundArgs a = {c, bounds, slots, count, __builtin_ctz((unsigned)c.page_size), (c.kv_heads + 3) / 4};
    const dim3 grid((unsigned)((count + kBoundSlots - 1) / kBoundSlots * a.head_blocks));
    if (c.bits == 8)
        ABQ_BOUND(8);
    else
        ABQ_BOUND(4);
    return hipGetLastError();
}

template <int D, int WAVES, bool SCORED> static hipError_t choose(const ChooseArgs &a, const uint32_t *scored, int64_t units, hipStream_t stream)
{
    const size_t lds = sizeof(uint32_t) * a.max_pages;
    if (lds > 48 << 10) { // (beyond what a launch gets unasked)
        const hipError_t e = hipFuncSetAttribute((const void *)attn_choose_kernel<D, WAVES, SCORED>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess)
            return e;
    }
    hipLaunchKernelGGL((attn_choose_kernel<D, WAVES, SCORED>), dim3((unsigned)units), dim3(64 * WAVES), lds, stream, a, scored);
    return hipGetLastError();
}

template <int D> static hipError_t choose(const ChooseArgs &a, int64_t units, int likely, uint32_t *scored, hipStream_t stream)
{
    if (scored) {
        const int parts = (a.max_pages + kScorePages - 1) / kScorePages;
        hipLaunchKernelGGL(attn_score_kernel<D>, dim3((unsigned)(units * parts)), dim3(64 * kScoreWaves), 0, stream, a, scored);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess)
            return e;
        return likely <= 1024 ? choose<D, 8, true>(a, scored, units, stream) : choose<D, 16, true>(a, scored, units, stream);
    }
    // Waves: enough to score all pages in a round of 64 a wave, but no more than leave two (eight waves) or four workgroups to a compute unit
    // where there are more of these than units.  128 channels, us with 4, 8, 16 waves: 32 of 125 pages 7.6, 7.9, 9.3; 128 of 512 13.9, 13.4, 14.3;
    // 256 of 1200 29, 25, 23; 280 of 1250 34, 30, 37; 512 of 1200 43, 38, 46; 2048 of 1000 82, 90, 133
    if (likely <= 256 || units > 512)
        return choose<D, 4, false>(a, nullptr, units, stream);
    return likely <= 512 || units > 256 ? choose<D, 8, false>(a, nullptr, units, stream) : choose<D, 16, false>(a, nullptr, units, stream);
}

// A launch of their own for the scores, where few workgroups would each have many: us in one launch and in two, 8 of 600 pages 12.5 and 10.3,
// of 1200 18.4 and 11.8, of 8000 84 and 28; 64 of 600 13.1 and 12.3, of 2500 33 and 23; but 8 of 300 9.2 and 9.6, 128 of 1200 20.5 and 20.9
size_t choose_workspace_bytes(int64_t units, int max_pages, int likely)
{
    return likely > 512 && units <= 64 ? (size_t)units * max_pages * sizeof(uint32_t) : 0;
}

hipError_t launch_attn_choose(const ChooseCall &call, hipStream_t stream)
{
    if (call.q.rows == 0)
        return hipSuccess;
    const ChooseArgs a = {call.cache, call.bounds, call.q, call.page_table, call.context, call.q_starts, call.blocks, call.dtype, call.heads / call.cache.kv_heads,
                          call.seqs, call.max_q, call.max_pages, call.first, call.last, call.count, __builtin_ctz((unsigned)call.cache.page_size)};
    const int64_t units = (int64_t)call.seqs * call.max_q * call.cache.kv_heads;
    const size_t need = choose_workspace_bytes(units, call.max_pages, call.likely);
    uint32_t *scored = need && call.workspace_bytes >= need ? (uint32_t *)call.workspace : nullptr;
    return call.cache.head_dim == 64 ? choose<64>(a, units, call.likely, scored, stream) : choose<128>(a, units, call.likely, scored, stream);
}

} // namespace abq
