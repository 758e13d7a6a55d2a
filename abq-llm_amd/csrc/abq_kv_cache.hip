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
#include "abq_kv_rows.h"

namespace abq {

namespace {

template <int DTYPE, int BITS, int D> __global__ __launch_bounds__(256) void kv_append_kernel(CacheArgs a)
{
    const int lane = threadIdx.x & 63, li = lane % (D / 8);
    int token, head;
    if (!place<D>(a, blockIdx.x, lane, &token, &head))
        return;
    const int from = min(token, a.tokens - 1);
    const uint4 k = *(const uint4 *)((const uint16_t *)a.k.data + (int64_t)from * a.k.row_stride + (int64_t)head * a.k.head_stride + 8 * li);
    const uint4 v = *(const uint4 *)((const uint16_t *)a.v.data + (int64_t)from * a.v.row_stride + (int64_t)head * a.v.head_stride + 8 * li);
    const int slot = token < a.tokens ? a.slots[from] : -1;
    const Place at = place_of(a, slot);
    const bool whole = whole_quad<D>(slot, lane);
    append_row<DTYPE, BITS, D, 0>(a, k, at, head, lane, whole);
    append_row<DTYPE, BITS, D, 1>(a, v, at, head, lane, whole);
}

template <int DTYPE, int BITS, int D> __global__ __launch_bounds__(256) void kv_read_kernel(CacheArgs a)
{
    constexpr int kLanes = D / 8;
    constexpr int R = D * BITS / 8;
    const int lane = threadIdx.x & 63, li = lane % kLanes;
    int token, head;
    if (!place<D>(a, blockIdx.x, lane, &token, &head) || token >= a.tokens)
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

} // namespace

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
