// Rotary positions: queries and keys turned by their tokens' positions, and the turned keys quantised into the cache on the way.
// The formulas are those stated in abq_attention.h.
//
// A wave takes one token (and some of its heads, where there are few tokens).  Its lanes work out the token's angles once, one pair each,
// and hand them round through LDS; then it goes over the heads.  A lane holds eight pairs, which are two pieces of eight elements of a
// row (i and i + rotary_dim / 2, or neighbours), so nothing crosses lanes but a row's extrema, and rows may be turned in place.
// The turned elements are fp64, whose products and sums this chip takes at the rate of fp32: two rows that differ by a last bit of
// fp32 may fall on either side of a code's border, and a cache that is filled token by token has to hold what one filled at once holds.
// Values, which four tokens share words of in the cache, are quantised by further workgroups of the same launch, as abq_kv_cache.hip does.
//
// Bound by memory: 16384 tokens of 32 + 32 heads of 128, fp16, turned, kept and quantised to 8 bits, 810 MB in 183 us, 4.4 TB/s where a
// copy reaches 5.0 (with fp32 instead of fp64 181, without scales 179, without the keys' quantisation 164); turned alone 104, 5.2 TB/s.  777
// tokens of 40 + 40 heads, bf16, 4 bits, 44 MB: 12.6, where turning and appending in two calls take 16.4.  16 tokens: 3.4, the launch and a
// chain of four loads.
#include "abq_kv_rows.h"
#include "abq_decoding.h"

#include <type_traits>

namespace abq {

namespace {

struct RotaryArgs {
    const double *turns;
    const int32_t *axis, *positions;
    int64_t position_stride;
    abq_rows q, q_out, k, k_out;
    int heads[2]; // of queries, of keys
    int pairs, axes;
    int tokens, splits; // splits: waves that share a token's heads
};

constexpr int kMostPairs = 128; // of a head of 256

// The lane's two pieces of eight elements: where they stand in the row, and whether they turn
struct Pieces {
    int e0, e1;
    bool turn;
};
__device__ __forceinline__ Pieces pieces_of(const RotaryArgs &r, bool beside, int chunk)
{
    const bool turn = 8 * chunk < r.pairs;
    const bool apart = turn && !beside;
    return {apart ? 8 * chunk : 16 * chunk, apart ? r.pairs + 8 * chunk : 16 * chunk + 8, turn};
}


// How far the position has turned, less whole turns: the product is rounded, as the formula says, and not contracted with what is taken off
__device__ __forceinline__ double part_of_turn(int position, double turns)
{
#pragma clang fp contract(off)
    const double t = (double)position * turns;
    return t - rint(t);
}

// Cosine and sine of f turns, |f| <= 1/2, from their Taylor series: the nearest quarter turn is taken off exactly, what is left is an eighth of a turn
// at most, and the first terms left out, x^17 / 17! and x^18 / 18!, are below 2^-54.
__device__ __forceinline__ double2 cos_sin(double f)
{
    const double quarter = rint(4 * f), x = (4 * f - quarter) * 1.57079632679489661923, y = x * x;
    double s = -1. / 1307674368000., c = 1. / 20922789888000.;
    constexpr double kSin[] = {1. / 6227020800., -1. / 39916800., 1. / 362880., -1. / 5040., 1. / 120., -1. / 6.};
    constexpr double kCos[] = {-1. / 87178291200., 1. / 479001600., -1. / 3628800., 1. / 40320., -1. / 720., 1. / 24., -1. / 2.};
#pragma unroll
    for (const double k : kSin)
        s = __builtin_fma(s, y, k);
#pragma unroll
    for (const double k : kCos)
        c = __builtin_fma(c, y, k);
    s = __builtin_fma(x * y, s, x);
    c = __builtin_fma(c, y, 1.);
    const int q = (int)quarter & 3; // (-2 .. 2: a half turn is either)
    const double a = q & 1 ? s : c, b = q & 1 ? c : s;
    return {q == 1 || q == 2 ? -a : a, q >= 2 ? -b : b};
}

// fp32, for good: the compiler would round fp64 to the type at once, in an emulation of some ten operations
__device__ __forceinline__ float rounded(double x)
{
    float y = (float)x;
    asm("" : "+v"(y));
    return y;
}

// Turns 16 elements.  The roundings are to fp32 and then to the type, as a conversion of fp64 is done here: the second one meets a
// tie that was none in one of 2^13 cases, and is then off by half a step as any rounding.
template <int DTYPE, bool BESIDE> __device__ __forceinline__ void turn16(uint4 &lo, uint4 &hi, const double (&c)[8], const double (&s)[8])
{
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    uint32_t y[8];
    if constexpr (BESIDE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double a = value16<DTYPE>(w[i]), b = value16<DTYPE>(w[i] >> 16);
            y[i] = pack16<DTYPE>(rounded(a * c[i] - b * s[i]), rounded(b * c[i] + a * s[i]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double a0 = value16<DTYPE>(w[i]), a1 = value16<DTYPE>(w[i] >> 16), b0 = value16<DTYPE>(w[4 + i]), b1 = value16<DTYPE>(w[4 + i] >> 16);
            y[i] = pack16<DTYPE>(rounded(a0 * c[2 * i] - b0 * s[2 * i]), rounded(a1 * c[2 * i + 1] - b1 * s[2 * i + 1]));
            y[4 + i] = pack16<DTYPE>(rounded(b0 * c[2 * i] + a0 * s[2 * i]), rounded(b1 * c[2 * i + 1] + a1 * s[2 * i + 1]));
        }
    }
    lo = uint4{y[0], y[1], y[2], y[3]};
    hi = uint4{y[4], y[5], y[6], y[7]};
}

// Quantises the row that the lane holds the elements e0 .. e0 + 7 and e1 .. e1 + 7 of, by D / 16 lanes, into the keys
template <int DTYPE, int BITS, int D> __device__ __forceinline__ void append_key(const CacheArgs &a, uint4 lo, uint4 hi, const Pieces &p, const Place &at, int head, bool first)
{
    constexpr int R = D * BITS / 8;
    constexpr int kHalf = 1 << (BITS - 1);
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
        x[i] = value16<DTYPE>(w[i / 2] >> (16 * (i & 1)));
    QuantRow q;
    if (a.c.symmetric) {
        float mx = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            mx = fmaxf(mx, fabsf(x[i]));
        q = quant_row_params(max_of_row<D / 16>(mx), 0.f, BITS, 1);
    } else {
        float mx = x[0], mn = -x[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) {
            mx = fmaxf(mx, x[i]);
            mn = fmaxf(mn, -x[i]);
        }
        q = quant_row_params(max_of_row<D / 16>(mx), -max_of_row<D / 16>(mn), BITS, 0);
    }
    uint32_t code[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
        code[i] = (quant_code_bits(x[i], q) ^ kHalf) & (2 * kHalf - 1);
    if (!at.there)
        return;
    const int64_t row = ((int64_t)at.page * a.c.kv_heads + head) * a.c.page_size;
    if (first)
        write_scale<BITS>(a, a.c.k_scales, row, at.t, q);
    uint8_t *dst = (uint8_t *)a.c.k_codes + (row + at.t) * R;
    write_key_codes<BITS>(dst, p.e0 / 8, code);
    write_key_codes<BITS>(dst, p.e1 / 8, code + 8);
}

// BESIDE: pairs are neighbours.  BITS 0: no cache.  Otherwise D is the head's size, and workgroups from `turning` on quantise values.
template <int DTYPE, int BITS, int D, bool BESIDE> __global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs r, CacheArgs a, int head_dim, uint32_t turning)
{
    __shared__ double2 angles[4][kMostPairs];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if constexpr (BITS != 0) {
        if (blockIdx.x >= turning) {
            int token, head;
            if (!place<D>(a, blockIdx.x - turning, lane, &token, &head))
                return;
            const int from = min(token, a.tokens - 1);
            const uint4 v = *(const uint4 *)((const uint16_t *)a.v.data + (int64_t)from * a.v.row_stride + (int64_t)head * a.v.head_stride + 8 * (lane % (D / 8)));
            const int slot = token < a.tokens ? a.slots[from] : -1;
            append_row<DTYPE, BITS, D, 1>(a, v, place_of(a, slot), head, lane, whole_quad<D>(slot, lane));
            return;
        }
    }
    const uint32_t unit = blockIdx.x * 4 + wave;
    const int token = unit / r.splits, split = unit % r.splits;
    if (token >= r.tokens)
        return;
    // (what a wave writes here it reads itself, in order: no barrier)
    for (int i = lane; i < r.pairs; i += 64) {
        const int axis = r.axis ? min(max(r.axis[i], 0), r.axes - 1) : 0;
        angles[wave][i] = cos_sin(part_of_turn(r.positions[axis * r.position_stride + token], r.turns[i]));
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int dim = BITS ? D : head_dim, lanes = dim / 16, rows = 64 / lanes; // lanes of a row, rows of a wave
    const int chunk = lane % lanes, mine = lane / lanes;
    const Pieces p = pieces_of(r, BESIDE, chunk);
    double c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double2 x = angles[wave][p.turn ? 8 * chunk + i : 0];
        c[i] = x.x;
        s[i] = x.y;
    }
    Place at = {};
    if constexpr (BITS != 0)
        at = place_of(a, a.slots[token]);
    // steps: rows of queries, then of keys
    const int steps_q = (r.heads[0] + rows - 1) / rows, steps = steps_q + (r.heads[1] + rows - 1) / rows;
    auto fetch = [&](int step, uint4 *lo, uint4 *hi) {
        const bool keys = step >= steps_q;
        const int head = (keys ? step - steps_q : step) * rows + mine;
        const uint16_t *src = (const uint16_t *)(keys ? r.k.data : r.q.data) + token * (keys ? r.k.row_stride : r.q.row_stride) +
                              (mine < rows && head < (keys ? r.heads[1] : r.heads[0]) ? head : 0) * (keys ? r.k.head_stride : r.q.head_stride);
        *lo = *(const uint4 *)(src + p.e0);
        *hi = *(const uint4 *)(src + p.e1);
    };
    auto turn = [&](uint4 lo0, uint4 hi0, const abq_rows &out, int heads, int step, auto keys) {
        const int head = step * rows + mine;
        uint4 lo = lo0, hi = hi0;
        turn16<DTYPE, BESIDE>(lo, hi, c, s);
        if (!p.turn) {
            lo.x = lo0.x, lo.y = lo0.y, lo.z = lo0.z, lo.w = lo0.w;
            hi.x = hi0.x, hi.y = hi0.y, hi.z = hi0.z, hi.w = hi0.w;
        }
        if (mine >= rows || head >= heads) // (a row's lanes are there together)
            return;
        if (out.data) {
            uint16_t *dst = (uint16_t *)out.data + token * out.row_stride + head * out.head_stride;
            *(uint4 *)(dst + p.e0) = lo;
            *(uint4 *)(dst + p.e1) = hi;
        }
        if constexpr (BITS != 0 && decltype(keys)::value)
            append_key<DTYPE, BITS, D>(a, lo, hi, p, at, head, chunk == 0);
    };
    int step = split;
    if (step >= steps)
        return;
    uint4 lo, hi, next_lo, next_hi;
    fetch(step, &lo, &hi);
    for (; step < steps; step += r.splits) {
        if (step + r.splits < steps) // (rows in place are read before any other is written: each is one lane's)
            fetch(step + r.splits, &next_lo, &next_hi);
        if (step < steps_q)
            turn(lo, hi, r.q_out, r.heads[0], step, std::false_type());
        else
            turn(lo, hi, r.k_out, r.heads[1], step - steps_q, std::true_type());
        lo = next_lo;
        hi = next_hi;
    }
}

} // namespace

// Waves that share a token's heads: enough of them for eight a compute unit (256 tokens of 32 + 8 heads 4.0 us, 777 of 40 + 40 12.6; with half as
// many 4.3 and 12.0, with four times as many 3.9 and 13.7)
int rotary_splits(int64_t tokens, int steps)
{
    const int64_t wanted = (2048 + tokens - 1) / (tokens > 0 ? tokens : 1);
    return (int)(wanted < 1 ? 1 : wanted < steps ? wanted : steps);
}

#define ABQ_ROTARY(T, B, D_)                                                                                               \
    do {                                                                                                                   \
        if (call.rotary.interleaved)                                                                                       \
            hipLaunchKernelGGL((rotary_kernel<T, B, D_, true>), grid, dim3(256), 0, stream, r, a, head_dim, turning);      \
        else                                                                                                               \
            hipLaunchKernelGGL((rotary_kernel<T, B, D_, false>), grid, dim3(256), 0, stream, r, a, head_dim, turning);     \
    } while (0)
#define ABQ_ROTARY_DIM(T, B)     \
    do {                         \
        if (head_dim == 64)      \
            ABQ_ROTARY(T, B, 64);  \
        else                     \
            ABQ_ROTARY(T, B, 128); \
    } while (0)

hipError_t launch_rotary(const RotaryCall &call, hipStream_t stream)
{
    RotaryArgs r;
    CacheArgs a = {};
    dim3 values(0);
    const int head_dim = call.head_dim, lanes = head_dim / 16, rows = 64 / lanes;
    r.turns = call.rotary.turns;
    r.axis = call.rotary.axis;
    r.positions = call.positions;
    r.position_stride = call.position_stride;
    r.pairs = call.rotary.rotary_dim / 2;
    r.axes = call.rotary.axes;
    r.q = call.q;
    r.q_out = call.q_out;
    r.k = call.k;
    r.k_out = call.k_out;
    r.heads[0] = call.heads[0];
    r.heads[1] = call.heads[1];
    if (call.tokens == 0)
        return hipSuccess;
    r.tokens = (int)call.tokens;
    r.splits = rotary_splits(call.tokens, (r.heads[0] + rows - 1) / rows + (r.heads[1] + rows - 1) / rows);
    const uint32_t turning = (uint32_t)((call.tokens * r.splits + 3) / 4);
    if (call.cache)
        cache_args(*call.cache, call.k, call.v, call.slots, &a, &values);
    const dim3 grid(turning + (call.cache ? values.x : 0));
    const bool bf16 = call.dtype == ABQ_BF16;
    if (!call.cache) {
        if (bf16)
            ABQ_ROTARY(ABQ_BF16, 0, 64);
        else
            ABQ_ROTARY(ABQ_F16, 0, 64);
    } else if (call.cache->bits == 8) {
        if (bf16)
            ABQ_ROTARY_DIM(ABQ_BF16, 8);
        else
            ABQ_ROTARY_DIM(ABQ_F16, 8);
    } else if (bf16)
        ABQ_ROTARY_DIM(ABQ_BF16, 4);
    else
        ABQ_ROTARY_DIM(ABQ_F16, 4);
    return hipGetLastError();
}

} // namespace abq
