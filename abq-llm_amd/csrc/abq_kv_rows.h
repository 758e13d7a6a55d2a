// Rows of new tokens on their way into the quantised cache: what its kernels (abq_kv_cache.hip) and those that turn the rows first
// (abq_rotary.hip) share on the device.  Layout and formulas are those stated in abq_attention.h.
#pragma once
#include "abq_attn.h"
#include "abq_quant.h"

namespace abq {

struct CacheArgs {
    abq_kv_cache c;
    abq_rows k, v;
    const int32_t *slots;
    int tokens, groups;  // groups: of the consecutive tokens that a wave holds
    int page_shift;
};
// and the workgroups of four waves that take them (abq_kv_cache.hip); false: no tokens
bool cache_args(const abq_kv_cache &c, const abq_rows &k, const abq_rows &v, const int32_t *slots, CacheArgs *a, dim3 *grid);

template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t x)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
template <int CTRL> __device__ __forceinline__ float max_dpp(float x)
{
    return fmaxf(x, __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(uint32_t, x))));
}
// over the 4, 8 or 16 lanes of a row: neighbours, pairs, for 8 the quads (mirrored halves), and for 16 the other eight
template <int LANES> __device__ __forceinline__ float max_of_row(float x)
{
    x = max_dpp<0x4e>(max_dpp<0xb1>(x));
    x = LANES >= 8 ? max_dpp<0x141>(x) : x;
    return LANES == 16 ? max_dpp<0x128>(x) : x;
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

// Where a token goes: page and offset of its slot, if that lies in the cache
struct Place {
    int page, t;
    bool there;
};
__device__ __forceinline__ Place place_of(const CacheArgs &a, int slot)
{
    const int page = slot >> a.page_shift;
    return {page, slot & (a.c.page_size - 1), slot >= 0 && page < a.c.num_pages};
}

// A row's scale and zero point as the cache keeps them; `row` is the head's first row in its page
template <int BITS> __device__ __forceinline__ void write_scale(const CacheArgs &a, float *scales, int64_t row, int t, const QuantRow &q)
{
    if (a.c.symmetric)
        scales[row + t] = q.scale;
    else {
        scales[2 * row + t] = q.scale;
        scales[2 * row + a.c.page_size + t] = q.zero_out + (float)(1 << (BITS - 1));
    }
}

// Eight codes of keys, elements 8 w .. 8 w + 7 of a row that starts at dst
template <int BITS> __device__ __forceinline__ void write_key_codes(uint8_t *dst, int w, const uint32_t *code)
{
    if (BITS == 8)
        *(uint2 *)(dst + 8 * w) =
            uint2{code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24, code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24};
    else // nibbles 0, 4, 1, 5, 2, 6, 3, 7
        *(uint32_t *)(dst + 4 * w) = code[0] | code[1] << 16 | code[2] << 4 | code[3] << 20 | code[4] << 8 | code[5] << 24 | code[6] << 12 | code[7] << 28;
}

// The lane's token and its wave's head, for workgroup `block` of those that hold rows of D / 8 lanes; heads come first, so that the waves
// of a workgroup read neighbouring heads of the same tokens.
template <int D> __device__ __forceinline__ bool place(const CacheArgs &a, uint32_t block, int lane, int *token, int *head)
{
    const uint32_t unit = block * 4 + (threadIdx.x >> 6), group = unit / a.c.kv_heads;
    *token = group * (512 / D) + lane / (D / 8);
    *head = unit % a.c.kv_heads;
    return group < (uint32_t)a.groups;
}

// Whether the lane's token is one of four of the wave that lie beside each other in the cache, as prompts do, so that their values are
// written as whole words
template <int D> __device__ __forceinline__ bool whole_quad(int slot, int lane)
{
    constexpr int kLanes = D / 8;
    const int first = __shfl(slot, (lane / (4 * kLanes)) * 4 * kLanes);
    const uint64_t wholes = __ballot((first & 3) == 0 && first >= 0 && slot == first + (lane / kLanes & 3));
    const uint64_t quad_lanes = D == 128 ? ~0ull : 0xffffffffull << (lane & 32);
    return (wholes & quad_lanes) == quad_lanes;
}

// Quantises the row that the lane holds eight elements of, of keys (KV 0) or values (1), and writes it
template <int DTYPE, int BITS, int D, int KV>
__device__ __forceinline__ void append_row(const CacheArgs &a, uint4 w, const Place &at, int head, int lane, bool whole)
{
    constexpr int kLanes = D / 8; // lanes of a row
    constexpr int R = D * BITS / 8;
    constexpr int kHalf = 1 << (BITS - 1);
    const int li = lane % kLanes, quad = lane / kLanes & 3;
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
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
        q = quant_row_params(max_of_row<D / 8>(mx), 0.f, BITS, 1);
    } else {
        float mx = x[0], mn = -x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            mx = fmaxf(mx, x[i]);
            mn = fmaxf(mn, -x[i]);
        }
        q = quant_row_params(max_of_row<D / 8>(mx), -max_of_row<D / 8>(mn), BITS, 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        code[i] = (quant_code_bits(x[i], q) ^ kHalf) & (2 * kHalf - 1);

    const int64_t row = ((int64_t)at.page * a.c.kv_heads + head) * a.c.page_size; // the head's first row in its page
    if (at.there && li == 0)
        write_scale<BITS>(a, KV ? a.c.v_scales : a.c.k_scales, row, at.t, q);
    if constexpr (KV == 0) {
        if (at.there)
            write_key_codes<BITS>((uint8_t *)a.c.k_codes + (row + at.t) * R, li, code);
    } else {
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
        uint8_t *dst = (uint8_t *)a.c.v_codes + (row + (at.t & ~3)) * R; // the four tokens' columns
        if (whole) {
#pragma unroll
            for (int j = 0; j < kCols / 4; ++j) {
                uint32_t word = transpose_bytes<D>(cols[j], quad);
                if (BITS == 4)
                    word = __builtin_amdgcn_perm(word, word, 0x03010200u);
                if (at.there)
                    *(uint32_t *)(dst + (c0 + 4 * j + quad) * 4) = word;
            }
        } else if (at.there) {
            const int byte = BITS == 8 ? at.t & 3 : (at.t & 1) << 1 | (at.t >> 1 & 1);
#pragma unroll
            for (int j = 0; j < kCols; ++j)
                dst[(c0 + j) * 4 + byte] = (uint8_t)(cols[j / 4] >> (8 * (j & 3)));
        }
    }
}

} // namespace abq
