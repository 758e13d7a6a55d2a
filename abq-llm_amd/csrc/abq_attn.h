// Internal interface between the host API of attention (abq_attention.hip) and its kernels (abq_kv_cache.hip,
// abq_attn_prompt.hip, abq_attn_tree.hip), and what those share on the device.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "abq_attention.h"

namespace abq {

abq_status hip_status(hipError_t e); // abq_api.hip: records the error for abq_last_hip_error

hipError_t launch_kv_append(const abq_kv_cache &c, const abq_rows &k, const abq_rows &v, int dtype, const int32_t *slots, hipStream_t stream);
hipError_t launch_kv_read(const abq_kv_cache &c, const abq_rows &k, const abq_rows &v, int dtype, const int32_t *slots, hipStream_t stream);
hipError_t launch_attn_prompt(const abq_attn_state &st, hipStream_t stream);
hipError_t launch_attn_tree(const abq_attn_state &st, hipStream_t stream);

// How the work is laid out, from sizes alone (host)
void plan_attn_prompt(abq_attn_state *st, int most_parts);
void plan_attn_tree(abq_attn_state *st, int most_parts);

// HIP counts the threads of a launch in 32 bits; workgroups have 256, where nothing else is said
constexpr int64_t kMostThreads = 0xffffffffll, kMostBlocks = kMostThreads / 256;

// Bytes of the parts' results: per query row and head, `parts` sums of head_dim floats and as many pairs (maximum, sum)
inline size_t attn_parts_bytes(const abq_attn_state &st, int parts)
{
    return parts < 2 ? 0 : (size_t)st.q.rows * st.heads * parts * (st.head_dim + 2) * sizeof(float);
}

// The parts' results of one state in its workspace
struct AttnParts {
    float *sums;   // [row][head][part][head_dim], relative to the part's own maximum
    float2 *stats; // [row][head][part]: maximum (in powers of two) and sum of weights; a sum of 0: the part saw nothing
    int parts;
};
inline AttnParts attn_parts(const abq_attn_state &st)
{
    float *sums = (float *)st.workspace;
    return {sums, (float2 *)(sums + (size_t)st.q.rows * st.heads * st.parts * st.head_dim), st.parts};
}
// out = the parts' results joined (abq_attn_tree.hip)
hipError_t launch_attn_join(const abq_attn_state &st, hipStream_t stream);

typedef __attribute__((ext_vector_type(2))) _Float16 half2v;
typedef __attribute__((ext_vector_type(8))) _Float16 half8v;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8v;
typedef __attribute__((ext_vector_type(4))) float float4v;
typedef __attribute__((ext_vector_type(16))) float float16v;

// 16-bit floats by their bits
__device__ __forceinline__ float bf16_value(uint32_t bits) { return __builtin_bit_cast(float, bits << 16); }
__device__ __forceinline__ float f16_value(uint32_t bits) { return (float)__builtin_bit_cast(_Float16, (uint16_t)bits); }
template <int DTYPE> __device__ __forceinline__ float value16(uint32_t bits)
{
    return DTYPE == ABQ_BF16 ? bf16_value(bits & 0xffff) : f16_value(bits & 0xffff);
}
// two floats rounded (half to even) to a pair of 16-bit ones, a in the low half
template <int DTYPE> __device__ __forceinline__ uint32_t pack16(float a, float b)
{
    if constexpr (DTYPE == ABQ_BF16) {
        typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2v;
        return __builtin_bit_cast(uint32_t, bf16x2v{(__bf16)a, (__bf16)b});
    } else
        return __builtin_bit_cast(uint32_t, half2v{(_Float16)a, (_Float16)b});
}

// A result that is finite, but beyond the type's largest, becomes that one: weights that were rounded on one side of a quotient alone
// take a mean of values at the end of the type past it
template <int DTYPE> __device__ __forceinline__ float largest16() { return DTYPE == ABQ_BF16 ? 0x1.fep127f : 65504.f; }
template <int DTYPE> __device__ __forceinline__ float saturated16(float x)
{
    return fabsf(x) < INFINITY ? __builtin_amdgcn_fmed3f(x, -largest16<DTYPE>(), largest16<DTYPE>()) : x;
}
template <int DTYPE> __device__ __forceinline__ uint32_t pack16_saturated(float a, float b) { return pack16<DTYPE>(saturated16<DTYPE>(a), saturated16<DTYPE>(b)); }

// Reductions over lanes l, l ^ 16, l ^ 32, l ^ 48 (over l, l ^ 32 alone: across_halves), the result in all of them.  A swap of a
// register with its own copy leaves one half's (or row's) values in the one and the other's in the other.
struct TwoWords {
    uint32_t a, b; // (words of their own: __builtin_bit_cast of an element of the builtin's result takes the first one)
};
__device__ __forceinline__ TwoWords swap_halves(float x)
{
    const uint32_t w = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return {r[0], r[1]};
}
__device__ __forceinline__ TwoWords swap_rows(float x)
{
    const uint32_t w = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    return {r[0], r[1]};
}
__device__ __forceinline__ float max_of(TwoWords r) { return fmaxf(__builtin_bit_cast(float, r.a), __builtin_bit_cast(float, r.b)); }
__device__ __forceinline__ float sum_of(TwoWords r) { return __builtin_bit_cast(float, r.a) + __builtin_bit_cast(float, r.b); }
__device__ __forceinline__ float max_across_halves(float x) { return max_of(swap_halves(x)); }
__device__ __forceinline__ float sum_across_halves(float x) { return sum_of(swap_halves(x)); }
__device__ __forceinline__ float max_across_quarters(float x) { return max_across_halves(max_of(swap_rows(x))); }
__device__ __forceinline__ float sum_across_quarters(float x) { return sum_across_halves(sum_of(swap_rows(x))); }

constexpr float kLog2e = 1.44269504088896340736f;

// A sequence's rows [first, first + count) of `rows`, whatever its offsets hold
struct SeqRows {
    int first, count;
};
__device__ __forceinline__ SeqRows seq_rows(const int32_t *starts, int s, int64_t rows)
{
    const int most = (int)(rows < 0x7fffffff ? rows : 0x7fffffff);
    const int a = min(max(starts[s], 0), most), b = min(max(starts[s + 1], a), most);
    return {a, b - a};
}

} // namespace abq
