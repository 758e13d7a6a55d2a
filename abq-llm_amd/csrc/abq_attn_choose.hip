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

// ---------------------------------------------------------------------------------------------------------- bounds

struct BoundArgs {
    abq_kv_cache c;
    abq_kv_bounds b;
    const int32_t *slots;
    int64_t count;
    int page_shift, head_blocks;
};

constexpr int kBoundSlots = 16; // that a workgroup looks through

// The elements of a lane's 16 bytes of codes, in order
template <int BITS> __device__ __forceinline__ float code_of(const uint32_t (&w)[4], int e)
{
    if (BITS == 8)
        return (float)(w[e / 4] >> (8 * (e & 3)) & 255);
    return (float)(w[e / 8] >> (4 * ((e & 1) * 4 + (e & 7) / 2)) & 15);
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
        float most = 0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
#pragma unroll
            for (int o = kLanes; o < 64; o *= 2) {
                hi[e] = fmaxf(hi[e], __shfl_xor(hi[e], o));
                lo[e] = fminf(lo[e], __shfl_xor(lo[e], o));
            }
            most = fmaxf(most, fmaxf(fabsf(hi[e]), fabsf(lo[e])));
        }
#pragma unroll
        for (int o = 1; o < kLanes; o *= 2)
            most = fmaxf(most, __shfl_xor(most, o));
        const QuantRow q = quant_row_params(most, 0.f, 8, 1);
        const int64_t at = (int64_t)page * a.c.kv_heads + head;
        if (lane == 0)
            a.b.scales[at] = q.scale;
        if (lane < kLanes) {
            int8_t *dst = a.b.codes + at * 2 * D + li * kEach;
#pragma unroll
            for (int e = 0; e < kEach; e += 4) {
                uint32_t h = 0, l = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    h |= (quant_code_bits(hi[e + k], q) & 255) << (8 * k);
                    l |= (quant_code_bits(lo[e + k], q) & 255) << (8 * k);
                }
                *(uint32_t *)(dst + e) = h;
                *(uint32_t *)(dst + D + e) = l;
            }
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

// Floats as unsigned numbers of the same order
__device__ __forceinline__ uint32_t ordered(float x)
{
    const uint32_t w = __builtin_bit_cast(uint32_t, x);
    return w & 0x80000000u ? ~w : w | 0x80000000u;
}

// A workgroup per query and key head: scores of all pages into LDS, the count-th largest of them by a search over its bits, and the pages
// from there on, in order.
template <int D, int WAVES> __global__ __launch_bounds__(64 * WAVES) void attn_choose_kernel(ChooseArgs a)
{
    extern __shared__ uint32_t keys[]; // [max_pages]
    __shared__ int32_t counted[2][WAVES][4];
    constexpr int kThreads = 64 * WAVES, kChunks = D / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = lane & 15, g = lane >> 4;
    const int head = blockIdx.x % a.c.kv_heads, draft = blockIdx.x / a.c.kv_heads % a.max_q, seq = blockIdx.x / a.c.kv_heads / a.max_q;
    const SeqRows own = seq_rows(a.q_starts, seq, a.q.rows);
    if (draft >= own.count)
        return;
    const int n = min(max(a.context[seq], 0) >> a.page_shift, a.max_pages), want = a.count;
    const int64_t q_row = own.first + draft;
    int32_t *out = a.blocks + (q_row * a.c.kv_heads + head) * want;
    if (n <= want) {
        for (int i = threadIdx.x; i < want; i += kThreads)
            out[i] = i < n ? i : -1;
        return;
    }
    const int32_t *pages = a.page_table + (int64_t)seq * a.max_pages;

    for (int h0 = 0; h0 < a.group; h0 += 16) {
        // heads h0 .. h0 + 15 as rows of the product: lane (t, g) has the channels 64 j + 16 g .. + 15 of head h0 + t
        const bool there = h0 + t < a.group;
        const uint16_t *src = (const uint16_t *)a.q.data + q_row * a.q.row_stride + (int64_t)(head * a.group + (there ? h0 + t : 0)) * a.q.head_stride + 16 * g;
        float x[kChunks][16], most = 0;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            const uint4 w0 = *(const uint4 *)(src + 64 * j), w1 = *(const uint4 *)(src + 64 * j + 8);
            const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t bits = w[i / 2] >> (16 * (i & 1));
                x[j][i] = a.dtype == ABQ_BF16 ? value16<ABQ_BF16>(bits) : value16<ABQ_F16>(bits);
                most = fmaxf(most, fabsf(x[j][i]));
            }
        }
        const QuantRow row = quant_row_params(max_across_quarters(most), 0.f, 8, 1);
        int4v up[kChunks], down[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t u = 0, d = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = (int8_t)quant_code_bits(x[j][4 * k + i], row);
                    u |= (uint32_t)max(c, 0) << (8 * i);
                    d |= (uint32_t)(min(c, 0) & 255) << (8 * i);
                }
                up[j][k] = (int)u;
                down[j][k] = (int)d;
            }
        float scale[4];
        bool heads[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            scale[i] = __shfl(row.scale, 4 * g + i);
            heads[i] = h0 + 4 * g + i < a.group;
        }
        for (int p0 = 16 * wave; p0 < n; p0 += 16 * WAVES) {
            const int p = min(p0 + t, n - 1), page = pages[p];
            const bool in_cache = (uint32_t)page < (uint32_t)a.c.num_pages;
            const int64_t at = (int64_t)(in_cache ? page : 0) * a.c.kv_heads + head;
            const int8_t *bound = a.b.codes + at * 2 * D + 16 * g;
            int4v acc = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(up[j], *(const int4v *)(bound + 64 * j), acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(down[j], *(const int4v *)(bound + D + 64 * j), acc, 0, 0, 0);
            }
            // (lane (t, g) has page t's sums of heads 4 g .. 4 g + 3)
            float score = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                score = heads[i] ? fmaxf(score, (float)acc[i] * scale[i]) : score;
            score = max_across_quarters(score);
            if (g == 0 && p0 + t < n) {
                if (h0 > 0)
                    score = fmaxf(score, __builtin_bit_cast(float, keys[p]));
                if (h0 + 16 < a.group)
                    keys[p] = __builtin_bit_cast(uint32_t, score);
                else
                    keys[p] = p < a.first || p >= n - a.last ? ~0u : in_cache ? ordered(score * a.b.scales[at]) : 0;
            }
        }
    }
    __syncthreads();

    // the largest number that at least `want` keys reach, two bits at a time; `exact`: reached by no more than those
    uint32_t least = 0;
    bool exact = false;
    for (int shift = 30, round = 0; shift >= 0 && !exact; shift -= 2, ++round) {
        int over[3] = {0, 0, 0};
        for (int i = threadIdx.x; i < (n + kThreads - 1) / kThreads * kThreads; i += kThreads) {
            const uint32_t key = i < n ? keys[i] : 0;
#pragma unroll
            for (int j = 0; j < 3; ++j)
                over[j] += __popcll(__ballot(i < n && key >= least + ((uint32_t)(j + 1) << shift)));
        }
        if (lane < 3)
            counted[round & 1][wave][lane] = lane == 0 ? over[0] : lane == 1 ? over[1] : over[2];
        __syncthreads();
        int total[3] = {0, 0, 0};
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
#pragma unroll
            for (int j = 0; j < 3; ++j)
                total[j] += counted[round & 1][w][j];
#pragma unroll
        for (int j = 2; j >= 0; --j)
            if (total[j] >= want) {
                least += (uint32_t)(j + 1) << shift;
                exact = total[j] == want;
                break;
            }
    }
    // How many of those that are just as large there is room for: all, or what the larger ones leave
    __syncthreads();
    int room = want;
    if (!exact) {
        int over = 0;
        for (int i = threadIdx.x; i < (n + kThreads - 1) / kThreads * kThreads; i += kThreads)
            over += __popcll(__ballot(i < n && keys[i] > least));
        if (lane == 0)
            counted[0][wave][0] = over;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
            room -= counted[0][w][0];
    }
    // in order: larger ones and equal ones before each page, in the two halves of a word (n < 2^16)
    uint32_t before = 0;
    for (int base = 0, round = 1; base < n; base += kThreads, ++round) {
        const int i = base + threadIdx.x;
        const uint32_t key = i < n ? keys[i] : 0;
        const bool larger = i < n && key > least, equal = i < n && key == least;
        const uint64_t l = __ballot(larger), e = __ballot(equal), below = (1ull << lane) - 1;
        uint32_t mine = __popcll(l & below) | __popcll(e & below) << 16;
        if (lane == 0)
            counted[round & 1][wave][3] = __popcll(l) | __popcll(e) << 16;
        __syncthreads();
        uint32_t all = before;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const uint32_t x = counted[round & 1][w][3];
            mine += w < wave ? x : 0;
            all += x;
        }
        mine += before;
        before = all;
        const int equal_before = mine >> 16, at = (mine & 0xffff) + min(equal_before, room);
        if (larger || (equal && equal_before < room))
            out[at] = i;
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

template <int D, int WAVES> static hipError_t choose(const ChooseArgs &a, dim3 grid, hipStream_t stream)
{
    const size_t lds = sizeof(uint32_t) * a.max_pages;
    if (lds > 48 << 10) { // (beyond what a launch gets unasked)
        const hipError_t e = hipFuncSetAttribute((const void *)attn_choose_kernel<D, WAVES>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess)
            return e;
    }
    hipLaunchKernelGGL((attn_choose_kernel<D, WAVES>), grid, dim3(64 * WAVES), lds, stream, a);
    return hipGetLastError();
}

hipError_t launch_attn_choose(const ChooseCall &call, hipStream_t stream)
{
    if (call.q.rows == 0)
        return hipSuccess;
    const ChooseArgs a = {call.cache, call.bounds, call.q, call.page_table, call.context, call.q_starts, call.blocks, call.dtype, call.heads / call.cache.kv_heads,
                          call.seqs, call.max_q, call.max_pages, call.first, call.last, call.count, __builtin_ctz((unsigned)call.cache.page_size)};
    const dim3 grid((unsigned)((int64_t)call.seqs * call.max_q * call.cache.kv_heads));
    return call.cache.head_dim == 64 ? choose<64, 8>(a, grid, stream) : choose<128, 8>(a, grid, stream);
}

} // namespace abq
