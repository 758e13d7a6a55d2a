// The quantised key / value cache: rows of new tokens quantised per token and head as they are written, and read back.
// The layout and the formulas are those stated in abq_attention.h.
//
// A row (64 or 128 elements) is held by 8 or 16 lanes, 8 elements each, so a wave holds 8 or 4 consecutive tokens of one head, and
// takes their keys and their values, requested together.  Extrema go over a row's lanes, and the four tokens that the values'
// layout puts beside each other change places, by lane permutes without LDS.
//
// Bound by memory: 2 bytes per element read and bits / 8 written, and the other way round when read back.  Keys and values of
// 16 x 1024 tokens of 32 heads of 128, 8 bits, 407 MB each way: 87 us written (4.7 TB/s), 69 us read back (5.9, some of it what
// was just written and is still on the chip), where a copy reaches 5.1.  One token for each of 16 sequences, 1 MB, is the launch: 4.3 and
// 2.8 us.
#include "abq_attn.h"
#include "abq_quant.h"

namespace abq {

namespace {

struct CacheArgs {
    abq_kv_cache c;
    abq_rows k, v;
    const int32_t *slots;
    int tokens, groups;  // groups: of the consecutive tokens that a wave holds
    int page_shift;
};

template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t x)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
template <int CTRL> __device__ __forceinline__ float max_dpp(float x)
{
    return fmaxf(x, __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(uint32_t, x))));
}
// over the 8 or 16 lanes of a row: neighbours, pairs, quads (mirrored halves), and for 16 the other eight
template <int D> __device__ __forceinline__ float max_of_row(float x)
{
    x = max_dpp<0x141>(max_dpp<0x4e>(max_dpp<0xb1>(x)));
    return D == 128 ? max_dpp<0x128>(x) : x;
}

// Columns 0 .. 3 of four tokens, one token's per lane (its bytes in `own`), dealt out so that the lane of token t gets column t
// with a token's byte in every place.  Tokens are D / 8 lanes apart.
template <int D> __device__ __forceinline__ uint32_t transpose_bytes(uint32_t own, int t)
{
    // an even token keeps columns 0 and 2 of the pair, an odd one 1 and 3 (v_perm_b32: bytes 0 - 3 of the second operand, 4 - 7 of the first)
    uint32_t pair;
    if constexpr (D == 128) {
        const auto r = __builtin_amdgcn_permlane16_swap(own, own, false, false);
        pair = __builtin_amdgcn_perm(r[1], r[0], t & 1 ? 0x07030501u : 0x06020400u);
    } else
        pair = __builtin_amdgcn_perm(dpp<0x128>(own), own, t & 1 ? 0x03070105u : 0x06020400u);
    const uint32_t columns = t & 2 ? 0x07060302u : 0x05040100u;
    if constexpr (D == 128) {
        const auto r = __builtin_amdgcn_permlane32_swap(pair, pair, false, false);
        return __builtin_amdgcn_perm(r[1], r[0], columns);
    } else {
        const auto r = __builtin_amdgcn_permlane16_swap(pair, pair, false, false);
        return __builtin_amdgcn_perm(r[1], r[0], columns);
    }
}

// The lane's token and its wave's head; heads come first, so that the waves of a workgroup read neighbouring heads of
// the same tokens.
template <int D> __device__ __forceinline__ bool place(const CacheArgs &a, int lane, int *token, int *head)
{
    const uint32_t unit = blockIdx.x * 4 + (threadIdx.x >> 6), group = unit / a.c.kv_heads;
    *token = group * (512 / D) + lane / (D / 8);
    *head = unit % a.c.kv_heads;
    return group < (uint32_t)a.groups;
}

template <int DTYPE, int BITS, int D> __global__ __launch_bounds__(256) void kv_append_kernel(CacheArgs a)
{
    constexpr int kLanes = D / 8; // lanes of a row
    constexpr int R = D * BITS / 8;
    constexpr int kHalf = 1 << (BITS - 1);
    const int lane = threadIdx.x & 63, li = lane % kLanes;
    int token, head;
    if (!place<D>(a, lane, &token, &head))
        return;
    const int from = min(token, a.tokens - 1);
    const uint4 w[2] = {*(const uint4 *)((const uint16_t *)a.k.data + (int64_t)from * a.k.row_stride + (int64_t)head * a.k.head_stride + 8 * li),
                        *(const uint4 *)((const uint16_t *)a.v.data + (int64_t)from * a.v.row_stride + (int64_t)head * a.v.head_stride + 8 * li)};
    const int slot = token < a.tokens ? a.slots[from] : -1;
    const bool there = slot >= 0 && (slot >> a.page_shift) < a.c.num_pages;
    const int page = slot >> a.page_shift, t = slot & (a.c.page_size - 1);
    // Four tokens of the wave that lie beside each other in the cache, as prompts do, have their values written as whole words.
    const int quad = lane / kLanes & 3;
    const int first = __shfl(slot, (lane / (4 * kLanes)) * 4 * kLanes);
    const uint64_t wholes = __ballot((first & 3) == 0 && first >= 0 && slot == first + quad);
    const uint64_t quad_lanes = D == 128 ? ~0ull : 0xffffffffull << (lane & 32);
    const bool whole = (wholes & quad_lanes) == quad_lanes;

#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        const uint32_t words[4] = {w[kv].x, w[kv].y, w[kv].z, w[kv].w};
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = value16<DTYPE>(words[i / 2] >> (16 * (i & 1)));
        uint32_t code[8];
        QuantRow q;
        if (a.c.symmetric) {
            float mx = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                mx = fmaxf(mx, fabsf(x[i]));
            q = quant_row_params(max_of_row<D>(mx), 0.f, BITS, 1);
        } else {
            float mx = x[0], mn = -x[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) {
                mx = fmaxf(mx, x[i]);
                mn = fmaxf(mn, -x[i]);
            }
            q = quant_row_params(max_of_row<D>(mx), -max_of_row<D>(mn), BITS, 0);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            code[i] = (quant_code_bits(x[i], q) ^ kHalf) & (2 * kHalf - 1);

        const int64_t row = ((int64_t)page * a.c.kv_heads + head) * a.c.page_size; // the head's first row in its page
        if (there && li == 0) {
            float *scales = kv ? a.c.v_scales : a.c.k_scales;
            if (a.c.symmetric)
                scales[row + t] = q.scale;
            else {
                scales[2 * row + t] = q.scale;
                scales[2 * row + a.c.page_size + t] = q.zero_out + (float)kHalf;
            }
        }
        if (kv == 0) {
            uint8_t *dst = (uint8_t *)a.c.k_codes + (row + t) * R;
            if (BITS == 8) {
                if (there)
                    *(uint2 *)(dst + 8 * li) = uint2{code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24,
                                                     code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24};
            } else if (there) // nibbles 0, 4, 1, 5, 2, 6, 3, 7
                *(uint32_t *)(dst + 4 * li) =
                    code[0] | code[1] << 16 | code[2] << 4 | code[3] << 20 | code[4] << 8 | code[5] << 24 | code[6] << 12 | code[7] << 28;
            continue;
        }
        // values: byte columns, four tokens beside each other
        constexpr int kCols = BITS == 8 ? 8 : 4; // columns of a lane
        uint32_t cols[2];
        int c0; // the lane's first column
        cols[0] = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
        cols[1] = code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24;
        if (BITS == 8)
            c0 = 8 * li;
        else {
            // a column holds elements d and d + D / 2: of the eight columns that this lane and its partner share, the lower
            // lane takes the first four
            const uint32_t low2 = __shfl_xor(cols[0], kLanes / 2), high2 = __shfl_xor(cols[1], kLanes / 2);
            const bool upper = li >= kLanes / 2;
            cols[0] = upper ? high2 | cols[1] << 4 : cols[0] | low2 << 4;
            c0 = 8 * (li % (kLanes / 2)) + (upper ? 4 : 0);
        }
        uint8_t *dst = (uint8_t *)a.c.v_codes + (row + (t & ~3)) * R; // the four tokens' columns
        if (whole) {
#pragma unroll
            for (int j = 0; j < kCols / 4; ++j) {
                uint32_t word = transpose_bytes<D>(cols[j], quad);
                if (BITS == 4)
                    word = __builtin_amdgcn_perm(word, word, 0x03010200u);
                if (there)
                    *(uint32_t *)(dst + (c0 + 4 * j + quad) * 4) = word;
            }
        } else if (there) {
            const int at = BITS == 8 ? t & 3 : (t & 1) << 1 | (t >> 1 & 1);
#pragma unroll
            for (int j = 0; j < kCols; ++j)
                dst[(c0 + j) * 4 + at] = (uint8_t)(cols[j / 4] >> (8 * (j & 3)));
        }
    }
}

template <int DTYPE, int BITS, int D> __global__ __launch_bounds__(256) void kv_read_kernel(CacheArgs a)
{
    constexpr int kLanes = D / 8;
    constexpr int R = D * BITS / 8;
    const int lane = threadIdx.x & 63, li = lane % kLanes;
    int token, head;
    if (!place<D>(a, lane, &token, &head) || token >= a.tokens)
        return;
    const int slot = a.slots[token];
    const bool there = slot >= 0 && (slot >> a.page_shift) < a.c.num_pages;
    const int page = there ? slot >> a.page_shift : 0, t = slot & (a.c.page_size - 1);
    const int c0 = BITS == 8 ? 8 * li : 8 * (li % (kLanes / 2)); // the first of the lane's eight columns of values
    const int64_t row = ((int64_t)page * a.c.kv_heads + head) * a.c.page_size;
    const uint8_t *k = (const uint8_t *)a.c.k_codes + (row + t) * R, *v = (const uint8_t *)a.c.v_codes + (row + (t & ~3)) * R + c0 * 4;
    const uint2 kw = BITS == 8 ? *(const uint2 *)(k + 8 * li) : uint2{*(const uint32_t *)(k + 4 * li), 0};
    const uint4 vw[2] = {*(const uint4 *)v, *(const uint4 *)(v + 16)}; // (the lanes of the neighbouring tokens read the same words)
    const int64_t at_scale = a.c.symmetric ? row + t : 2 * row + t;
    const float scale[2] = {a.c.k_scales[at_scale], a.c.v_scales[at_scale]};
    float zero[2] = {(float)(1 << (BITS - 1)), (float)(1 << (BITS - 1))};
    if (!a.c.symmetric) {
        zero[0] = a.c.k_scales[at_scale + a.c.page_size];
        zero[1] = a.c.v_scales[at_scale + a.c.page_size];
    }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        uint32_t code[8];
        if (kv == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                code[i] = BITS == 8 ? (i < 4 ? kw.x : kw.y) >> (8 * (i & 3)) & 255 : kw.x >> (16 * (i & 1) + 4 * (i / 2)) & 15;
        } else {
            const uint32_t w[8] = {vw[0].x, vw[0].y, vw[0].z, vw[0].w, vw[1].x, vw[1].y, vw[1].z, vw[1].w};
            const int at = BITS == 8 ? 8 * (t & 3) : 8 * ((t & 1) << 1 | (t >> 1 & 1)) + (li >= kLanes / 2 ? 4 : 0);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                code[i] = w[i] >> at & ((1 << BITS) - 1);
        }
        uint32_t out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t two = pack16<DTYPE>(((float)code[2 * i] - zero[kv]) * scale[kv], ((float)code[2 * i + 1] - zero[kv]) * scale[kv]);
            out[i] = there ? two : 0;
        }
        const abq_rows &dst = kv ? a.v : a.k;
        *(uint4 *)((uint16_t *)dst.data + (int64_t)token * dst.row_stride + (int64_t)head * dst.head_stride + 8 * li) = uint4{out[0], out[1], out[2], out[3]};
    }
}

bool cache_args(const abq_kv_cache &c, const abq_rows &k, const abq_rows &v, const int32_t *slots, CacheArgs *a, dim3 *grid)
{
    a->c = c;
    a->k = k;
    a->v = v;
    a->slots = slots;
    a->tokens = (int)k.rows;
    const int rows = 512 / c.head_dim;
    a->groups = (a->tokens + rows - 1) / rows;
    a->page_shift = __builtin_ctz((unsigned)c.page_size);
    *grid = dim3((unsigned)(((int64_t)a->groups * c.kv_heads + 3) / 4));
    return a->tokens > 0;
}

} // namespace

#define ABQ_KV_CASES(KERNEL)                                                                  \
    do {                                                                                      \
        if (dtype == ABQ_BF16) {                                                              \
            if (c.bits == 8)                                                                  \
                ABQ_KV_DIM(KERNEL, ABQ_BF16, 8);                                              \
            else                                                                              \
                ABQ_KV_DIM(KERNEL, ABQ_BF16, 4);                                              \
        } else if (c.bits == 8)                                                               \
            ABQ_KV_DIM(KERNEL, ABQ_F16, 8);                                                   \
        else                                                                                  \
            ABQ_KV_DIM(KERNEL, ABQ_F16, 4);                                                   \
    } while (0)
#define ABQ_KV_DIM(KERNEL, T, B)                                                              \
    do {                                                                                      \
        if (c.head_dim == 64)                                                                 \
            hipLaunchKernelGGL((KERNEL<T, B, 64>), grid, dim3(256), 0, stream, a);            \
        else                                                                                  \
            hipLaunchKernelGGL((KERNEL<T, B, 128>), grid, dim3(256), 0, stream, a);           \
    } while (0)

hipError_t launch_kv_append(const abq_kv_cache &c, const abq_rows &k, const abq_rows &v, int dtype, const int32_t *slots, hipStream_t stream)
{
    CacheArgs a;
    dim3 grid;
    if (!cache_args(c, k, v, slots, &a, &grid))
        return hipSuccess;
    ABQ_KV_CASES(kv_append_kernel);
    return hipGetLastError();
}

hipError_t launch_kv_read(const abq_kv_cache &c, const abq_rows &k, const abq_rows &v, int dtype, const int32_t *slots, hipStream_t stream)
{
    CacheArgs a;
    dim3 grid;
    if (!cache_args(c, k, v, slots, &a, &grid))
        return hipSuccess;
    ABQ_KV_CASES(kv_read_kernel);
    return hipGetLastError();
}

} // namespace abq
