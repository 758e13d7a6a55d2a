// The quantised key / value cache: rows of new tokens quantised per token and head as they are written, and read back.
// The layout and the formulas are those stated in abq_attention.h.
//
// A row (64 or 128 elements) is held by 8 or 16 lanes, 8 elements each, so a wave holds 8 or 4 rows: consecutive tokens of one
// head, of the keys or of the values.  Extrema go over the row's lanes by shuffles; everything is read and written once.
// Bound by memory: 2 bytes per element read and bits / 8 written (and the other way round when read back).
#include "abq_attn.h"
#include "abq_quant.h"

namespace abq {

namespace {

struct CacheArgs {
    abq_kv_cache c;
    abq_rows k, v;
    const int32_t *slots;
    int tokens, groups; // groups: of the consecutive tokens that a wave holds
    int page_shift;
};

// Where a wave stands: which tokens, which head, keys or values.  Heads come first, so that the waves of a workgroup read
// neighbouring heads of the same tokens.
struct Place {
    int token, head, kv;
};

template <int D> __device__ __forceinline__ bool place(const CacheArgs &a, int lane, Place *p)
{
    constexpr int kRows = 512 / D;
    const uint32_t unit = blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t heads = 2 * a.c.kv_heads, group = unit / heads, rest = unit % heads;
    if (group >= (uint32_t)a.groups)
        return false;
    p->token = group * kRows + lane / (D / 8);
    p->head = rest % a.c.kv_heads;
    p->kv = rest / a.c.kv_heads;
    return true;
}

// Columns 0 .. 3 of four tokens, one token's per lane (its bytes in `own`), dealt out so that the lane of token t gets column t
// with a token's byte in every place.  `stride`: lanes between one token and the next.
__device__ __forceinline__ uint32_t transpose_bytes(uint32_t own, int t, int stride)
{
    const uint32_t other = __shfl_xor(own, stride);
    // an even token keeps columns 0 and 2 of the pair, an odd one 1 and 3 (v_perm_b32: bytes 0 - 3 of the second operand, 4 - 7 of the first)
    const uint32_t pair = t & 1 ? __builtin_amdgcn_perm(own, other, 0x07030501u) : __builtin_amdgcn_perm(other, own, 0x06020400u);
    const uint32_t far = __shfl_xor(pair, 2 * stride);
    return t & 2 ? __builtin_amdgcn_perm(pair, far, 0x07060302u) : __builtin_amdgcn_perm(far, pair, 0x05040100u);
}

template <int DTYPE, int BITS, int D> __global__ __launch_bounds__(256) void kv_append_kernel(CacheArgs a)
{
    constexpr int kLanes = D / 8; // lanes of a row
    constexpr int R = D * BITS / 8;
    const int lane = threadIdx.x & 63, li = lane % kLanes;
    Place p;
    if (!place<D>(a, lane, &p))
        return;
    const abq_rows &src = p.kv ? a.v : a.k;
    const bool mine = p.token < a.tokens;
    const int slot = mine ? a.slots[p.token] : -1;
    const bool there = slot >= 0 && (slot >> a.page_shift) < a.c.num_pages;
    uint4 w = {0, 0, 0, 0};
    if (there)
        w = *(const uint4 *)((const uint16_t *)src.data + (int64_t)p.token * src.row_stride + (int64_t)p.head * src.head_stride + 8 * li);
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] = value16<DTYPE>(words[i / 2] >> (16 * (i & 1)));
    float mx = x[0], mn = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        mx = fmaxf(mx, x[i]);
        mn = fminf(mn, x[i]);
    }
#pragma unroll
    for (int o = 1; o < kLanes; o *= 2) {
        mx = fmaxf(mx, __shfl_xor(mx, o));
        mn = fminf(mn, __shfl_xor(mn, o));
    }
    const QuantRow q = quant_row_params(mx, mn, BITS, a.c.symmetric);
    constexpr int kHalf = 1 << (BITS - 1);
    uint32_t code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        code[i] = (uint32_t)(quant_code(x[i], q) + kHalf) & (2 * kHalf - 1);

    const int page = slot >> a.page_shift, t = slot & (a.c.page_size - 1);
    const int64_t row = ((int64_t)page * a.c.kv_heads + p.head) * a.c.page_size; // the head's first row in its page
    if (there && li == 0) {
        float *scales = p.kv ? a.c.v_scales : a.c.k_scales;
        if (a.c.symmetric)
            scales[row + t] = q.scale;
        else {
            scales[2 * row + t] = q.scale;
            scales[2 * row + a.c.page_size + t] = q.zero_out + (float)kHalf;
        }
    }
    if (!p.kv) {
        uint8_t *dst = (uint8_t *)a.c.k_codes + (row + t) * R;
        if (BITS == 8) {
            const uint2 bytes = {code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24, code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24};
            if (there)
                *(uint2 *)(dst + 8 * li) = bytes;
        } else if (there) // nibbles 0, 4, 1, 5, 2, 6, 3, 7
            *(uint32_t *)(dst + 4 * li) = code[0] | code[1] << 16 | code[2] << 4 | code[3] << 20 | code[4] << 8 | code[5] << 24 | code[6] << 12 | code[7] << 28;
        return;
    }
    // values: byte columns, four tokens beside each other
    constexpr int kCols = BITS == 8 ? 8 : 4; // columns of a lane
    uint32_t cols[kCols / 4];
    int c0; // the lane's first column
    if (BITS == 8) {
        cols[0] = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
        cols[kCols / 4 - 1] = code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24;
        c0 = 8 * li;
    } else {
        // a column holds elements d and d + D / 2: of the eight columns that this lane and its partner share, the lower lane
        // takes the first four
        const uint32_t low = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24, high = code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24;
        const uint32_t low2 = __shfl_xor(low, kLanes / 2), high2 = __shfl_xor(high, kLanes / 2);
        const bool upper = li >= kLanes / 2;
        cols[0] = upper ? high2 | high << 4 : low | low2 << 4;
        c0 = 8 * (li % (kLanes / 2)) + (upper ? 4 : 0);
    }
    uint8_t *dst = (uint8_t *)a.c.v_codes + (row + (t & ~3)) * R; // the four tokens' columns
    // Four tokens of the wave that lie beside each other in the cache, as prompts do, are written as whole words.
    const int quad = lane / kLanes & 3;
    const int first = __shfl(slot, (lane / (4 * kLanes)) * 4 * kLanes);
    const bool whole = (first & 3) == 0 && first >= 0 && slot == first + quad;
    const uint64_t wholes = __ballot(whole);
    const uint64_t quad_lanes = D == 128 ? ~0ull : 0xffffffffull << (lane & 32);
    if ((wholes & quad_lanes) == quad_lanes) {
#pragma unroll
        for (int j = 0; j < kCols / 4; ++j) {
            uint32_t word = transpose_bytes(cols[j], quad, kLanes);
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

template <int DTYPE, int BITS, int D> __global__ __launch_bounds__(256) void kv_read_kernel(CacheArgs a)
{
    constexpr int kLanes = D / 8;
    constexpr int R = D * BITS / 8;
    const int lane = threadIdx.x & 63, li = lane % kLanes;
    Place p;
    if (!place<D>(a, lane, &p) || p.token >= a.tokens)
        return;
    const abq_rows &dst = p.kv ? a.v : a.k;
    uint4 *to = (uint4 *)((uint16_t *)dst.data + (int64_t)p.token * dst.row_stride + (int64_t)p.head * dst.head_stride + 8 * li);
    const int slot = a.slots[p.token], page = slot >> a.page_shift, t = slot & (a.c.page_size - 1);
    if (slot < 0 || page >= a.c.num_pages) {
        *to = uint4{0, 0, 0, 0};
        return;
    }
    const int64_t row = ((int64_t)page * a.c.kv_heads + p.head) * a.c.page_size;
    const float *scales = p.kv ? a.c.v_scales : a.c.k_scales;
    const float scale = scales[a.c.symmetric ? row + t : 2 * row + t];
    const float zero = a.c.symmetric ? (float)(1 << (BITS - 1)) : scales[2 * row + a.c.page_size + t];
    uint32_t code[8];
    if (!p.kv) {
        const uint8_t *src = (const uint8_t *)a.c.k_codes + (row + t) * R;
        if (BITS == 8) {
            const uint2 w = *(const uint2 *)(src + 8 * li);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                code[i] = (i < 4 ? w.x : w.y) >> (8 * (i & 3)) & 255;
        } else {
            const uint32_t w = *(const uint32_t *)(src + 4 * li);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                code[i] = w >> (16 * (i & 1) + 4 * (i / 2)) & 15;
        }
    } else {
        // the words of this lane's eight columns: the lanes of the neighbouring tokens read the same ones
        const uint8_t *src = (const uint8_t *)a.c.v_codes + (row + (t & ~3)) * R;
        const int c0 = BITS == 8 ? 8 * li : 8 * (li % (kLanes / 2));
        const uint4 w0 = *(const uint4 *)(src + c0 * 4), w1 = *(const uint4 *)(src + c0 * 4 + 16);
        const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
        const int at = BITS == 8 ? 8 * (t & 3) : 8 * ((t & 1) << 1 | (t >> 1 & 1)) + (li >= kLanes / 2 ? 4 : 0);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            code[i] = w[i] >> at & ((1 << BITS) - 1);
    }
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        out[i] = pack16<DTYPE>(((float)code[2 * i] - zero) * scale, ((float)code[2 * i + 1] - zero) * scale);
    *to = uint4{out[0], out[1], out[2], out[3]};
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
    *grid = dim3((unsigned)(((int64_t)a->groups * 2 * c.kv_heads + 3) / 4));
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
