// Which pages hold which sequence's tokens: tables that fork, grow and shrink on the device, and copies of pages.
// The rules are those stated in abq_attention.h; whole numbers throughout, and no result depends on the order of atomics (they only add).
//
// Tables are small (512 sequences of 40 pages, 80 KB; 6000 counts, 24 KB), so these calls are bound by launches and by the length of
// their chains of loads: whatever has to be decided in order is decided by one workgroup of 1024 threads that scans, everything
// else by as many as there is work for.  In a captured graph, 4 (512) sequences: fork 2.5 (4.1) us, growth by a token or taking it back 4.9
// (7.2); 4000 pages of 60 sequences made compact 9.7, of which the moves 5.8 and the entries' new names 3.9.  The workgroup that scans
// walks over a pool's occupied front in turns of 4096 pages, each of which waits for the last: 64 pages from behind 3600 occupied ones 9, from behind
// 54000 20, from behind 225000 54; 60000 pages made compact 65, 250000 250.
// Copies are bound by memory: 915 pages of 132 KB 46 to 49 us, 4.9 TB/s and more, the rate of any copy; pairs that copy nothing cost their workgroups'
// launch, 512 of them 5.2, 2000 16.
#include "abq_decoding.h"

namespace abq {

namespace {

struct PagesArgs {
    int32_t *table, *lengths, *refs;
    int seqs, max_pages, num_pages, page_shift;
};

__device__ __forceinline__ bool is_page(const PagesArgs &a, int32_t p) { return (uint32_t)p < (uint32_t)a.num_pages; }
__device__ __forceinline__ int pages_of(const PagesArgs &a, int tokens) { return (int)(((int64_t)tokens + (1 << a.page_shift) - 1) >> a.page_shift); }
// A length as it may be, whatever the array holds
__device__ __forceinline__ int length_of(const PagesArgs &a, int s)
{
    return (int)min((int64_t)max(a.lengths[s], 0), (int64_t)a.max_pages << a.page_shift);
}

// ---------------------------------------------------------------------------------------------------------- fork

// A workgroup takes `columns` columns of the whole table through LDS, so that rows may change places; one more takes the lengths.
__global__ __launch_bounds__(1024) void pages_fork_kernel(PagesArgs a, const int32_t *parents, int columns, int column_shift)
{
    extern __shared__ int32_t held[]; // [seqs][columns]
    const bool lengths = blockIdx.x == gridDim.x - 1;
    const int c0 = blockIdx.x * columns, shift = lengths ? 0 : column_shift, cells = a.seqs << shift;
    int32_t *at = lengths ? a.lengths : a.table + c0;
    const int64_t stride = lengths ? 1 : a.max_pages;
    const int last = lengths ? 1 : min(columns, a.max_pages - c0);
    for (int i = threadIdx.x; i < cells; i += 1024) {
        const int s = i >> shift, j = i & ((1 << shift) - 1);
        if (j < last)
            held[i] = at[s * stride + j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < cells; i += 1024) {
        const int s = i >> shift, j = i & ((1 << shift) - 1);
        if (j >= last)
            continue;
        const int parent = parents[s];
        const bool some = (uint32_t)parent < (uint32_t)a.seqs;
        const int32_t was = held[i], is = some ? held[(parent << shift) + j] : lengths ? 0 : -1;
        if (is == was)
            continue;
        at[s * stride + j] = is;
        if (!lengths) {
            if (is_page(a, was))
                atomicSub(&a.refs[was], 1);
            if (is_page(a, is))
                atomicAdd(&a.refs[is], 1);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------- extend

constexpr int kScan = 1024; // threads of the workgroup that scans

// The sum of x over the threads before this one, and over all; `sums` is LDS for the waves' own, not to be written again before a barrier
template <typename T> __device__ __forceinline__ T scan(T x, T *sums, T *total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T upto = x;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const T below = __shfl_up(upto, o);
        upto += lane >= o ? below : 0;
    }
    if (lane == 63)
        sums[wave] = upto;
    __syncthreads();
    const T of_wave = lane < kScan / 64 ? sums[lane] : 0;
    T before = of_wave;
#pragma unroll
    for (int o = 1; o < kScan / 64; o *= 2) {
        const T below = __shfl_up(before, o);
        before += lane >= o ? below : 0;
    }
    *total = __shfl(before, kScan / 64 - 1);
    return upto - x + __shfl(before - of_wave, wave);
}

// What a sequence asks for
struct Wish {
    int length, grow, shrink;
    int64_t pages; // that it needs
    bool fits, copied;
    int32_t last; // the page that its next token goes to, if that holds some of its tokens
};
__device__ __forceinline__ Wish wish_of(const PagesArgs &a, const int32_t *counts, int s)
{
    Wish w;
    const int count = counts[s];
    w.length = length_of(a, s);
    w.grow = max(count, 0);
    w.shrink = count < 0 ? (int)min(-(int64_t)count, (int64_t)w.length) : 0;
    const int64_t used = pages_of(a, w.length), wanted = ((int64_t)w.length + w.grow + (1 << a.page_shift) - 1) >> a.page_shift;
    w.fits = wanted <= a.max_pages;
    w.last = -1;
    w.copied = false;
    if (w.grow > 0 && w.fits && (w.length & ((1 << a.page_shift) - 1))) {
        w.last = a.table[(int64_t)s * a.max_pages + (w.length >> a.page_shift)];
        w.copied = is_page(a, w.last) && a.refs[w.last] > 1;
    }
    w.pages = w.grow > 0 && w.fits ? wanted - used + w.copied : 0;
    return w;
}

// The first sequence whose pages end behind number r of those handed out
__device__ __forceinline__ int owner_of(const int32_t *ends, int seqs, int r)
{
    int lo = 0, hi = seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > r)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo;
}

// The last sequence that starts at or before the row, of starts[0 .. seqs] with the row in front of the last
__device__ __forceinline__ int sequence_of(const int32_t *starts, int seqs, int64_t row)
{
    int lo = 0, hi = seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (starts[mid] <= row)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}
__device__ __forceinline__ int slot_of(const PagesArgs &a, int s, int place)
{
    return (a.table[(int64_t)s * a.max_pages + (place >> a.page_shift)] << a.page_shift) + (place & ((1 << a.page_shift) - 1));
}

// Page number j of a sequence that has become shorter
__device__ __forceinline__ void release(const PagesArgs &a, int s, int j)
{
    int32_t *entry = a.table + (int64_t)s * a.max_pages + j;
    if (is_page(a, *entry))
        atomicSub(&a.refs[*entry], 1);
    *entry = -1;
}

struct ExtendArgs {
    PagesArgs p;
    const int32_t *counts;
    int32_t *slots, *starts, *granted, *copies;
    int64_t rows;
};

// Everything that is decided in order, each sequence a thread's.  `all`: also what the second launch would do.
__global__ __launch_bounds__(kScan) void pages_extend_kernel(ExtendArgs e, int all)
{
    const PagesArgs &a = e.p;
    __shared__ int32_t ends[kMostSeqs]; // of the pages that sequences 0 .. s need, capped at kCapped
    __shared__ int32_t starts[kMostSeqs], lengths[kMostSeqs]; // of their new tokens; before the call
    __shared__ uint8_t flags[kMostSeqs];
    __shared__ int64_t sums[2][2][kScan / 64];
    __shared__ int32_t counted[2][kScan / 64];
    constexpr int32_t kCapped = 0x7fffffff; // (more than there can be pages)
    constexpr int kCopied = 1, kNeeds = 2, kGrows = 4, kGiven = 8, kShrinks = 16;
    // (the first pages' counts are asked for ahead of everything that waits for something else)
    const bool wide = ((uintptr_t)a.refs & 15) == 0;
    auto counts_of = [&](int p0) {
        if (wide && p0 + 3 < a.num_pages)
            return *(const int4 *)(a.refs + p0);
        return int4{p0 < a.num_pages ? a.refs[p0] : 1, p0 + 1 < a.num_pages ? a.refs[p0 + 1] : 1, p0 + 2 < a.num_pages ? a.refs[p0 + 2] : 1,
                    p0 + 3 < a.num_pages ? a.refs[p0 + 3] : 1};
    };
    int4 refs = counts_of(4 * threadIdx.x);
    int64_t all_need = 0, all_grow = 0;
    for (int s0 = 0, round = 0; s0 < a.seqs; s0 += kScan, ++round) {
        const int s = s0 + threadIdx.x;
        Wish w = {};
        if (s < a.seqs)
            w = wish_of(a, e.counts, s);
        int64_t here_need, here_grow;
        const int64_t need = all_need + scan(w.pages, sums[round & 1][0], &here_need), grow = all_grow + scan((int64_t)w.grow, sums[round & 1][1], &here_grow);
        if (s < a.seqs) {
            ends[s] = (int32_t)min(need + w.pages, (int64_t)kCapped);
            starts[s] = e.starts[s] = (int32_t)min(grow, (int64_t)kCapped);
            lengths[s] = w.length;
            flags[s] = (w.copied ? kCopied : 0) | (w.pages > 0 ? kNeeds : 0) | (w.grow > 0 && w.fits ? kGrows : 0);
            if (w.copied)
                e.copies[2 * s] = w.last;
        }
        all_need += here_need;
        all_grow += here_grow;
    }
    const int tokens = (int)min(all_grow, (int64_t)kCapped);
    if (threadIdx.x == 0)
        e.starts[a.seqs] = tokens;
    __syncthreads();
    // Free pages, in order, as the next ones of the sequences, until there are enough or no more.  One sequence at most gets only a
    // part of its pages, and gives them back below.
    const int64_t wanted = min(all_need, (int64_t)a.num_pages);
    int found = 0;
    for (int base = 0, round = 0; base < a.num_pages && found < wanted; base += 4 * kScan, ++round) {
        const int p0 = base + 4 * threadIdx.x;
        if (round > 0)
            refs = counts_of(p0);
        const bool free[4] = {refs.x == 0, refs.y == 0, refs.z == 0, refs.w == 0};
        int32_t here;
        int r = found + scan((int32_t)free[0] + free[1] + free[2] + free[3], counted[round & 1], &here);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!free[i] || r >= wanted)
                continue;
            const int s = owner_of(ends, a.seqs, r);
            const int64_t column = (int64_t)pages_of(a, lengths[s]) - (flags[s] & kCopied) + r - (s ? ends[s - 1] : 0);
            if (ends[s] < kCapped && column < a.max_pages) {
                a.table[(int64_t)s * a.max_pages + column] = p0 + i;
                a.refs[p0 + i] = 1;
            }
            ++r;
        }
        found += here;
    }
    __syncthreads();
    for (int s = threadIdx.x; s < a.seqs; s += kScan) {
        const int length = lengths[s], count = e.counts[s], first = s ? ends[s - 1] : 0, f = flags[s];
        const int64_t column = (int64_t)pages_of(a, length) - (f & kCopied);
        int32_t *entry = a.table + (int64_t)s * a.max_pages + column;
        const bool given = (f & kGrows) && (!(f & kNeeds) || ends[s] <= found);
        const int32_t from = f & kCopied ? e.copies[2 * s] : -1;
        if (!given && (f & kNeeds) && ends[s] < kCapped) // what it got, if anything, goes back
            for (int r = first; r < min(found, ends[s]); ++r) {
                if (is_page(a, entry[r - first]))
                    a.refs[entry[r - first]] = 0;
                entry[r - first] = r == first ? from : -1; // (from is -1 where nothing was to be copied)
            }
        if (given && (f & kCopied))
            atomicSub(&a.refs[from], 1);
        e.copies[2 * s] = given ? from : -1;
        e.copies[2 * s + 1] = given && (f & kCopied) ? *entry : -1;
        const int granted = given ? count : count < 0 ? -(int)min(-(int64_t)count, (int64_t)length) : 0;
        e.granted[s] = granted;
        a.lengths[s] = length + granted;
        if (all && granted < 0) {
            const int to = pages_of(a, length), kept = pages_of(a, length + granted);
            if (to - kept <= 4)
                for (int j = kept; j < to; ++j)
                    release(a, s, j);
            else
                flags[s] = kShrinks;
        } else if (all && given)
            flags[s] = kGiven;
    }
    if (!all)
        return;
    __syncthreads();
    for (int64_t row = threadIdx.x; row < e.rows; row += kScan) {
        int slot = -1;
        if (row < tokens) {
            const int s = sequence_of(starts, a.seqs, row);
            if (flags[s] == kGiven)
                slot = slot_of(a, s, lengths[s] + (int)(row - starts[s]));
        }
        e.slots[row] = slot;
    }
    // sequences that have lost many pages, a wave each
    const int lane = threadIdx.x & 63;
    for (int s0 = threadIdx.x & ~63; s0 < a.seqs; s0 += kScan) {
        const int s1 = s0 + lane;
        uint64_t many = __ballot(s1 < a.seqs && flags[min(s1, a.seqs - 1)] == kShrinks);
        for (; many; many &= many - 1) {
            const int s = s0 + __builtin_ctzll(many), to = pages_of(a, lengths[s]);
            for (int j = pages_of(a, a.lengths[s]) + lane; j < to; j += 64)
                release(a, s, j);
        }
    }
}

// What follows from it: slots, and the pages of sequences that have become shorter, a wave each, by the workgroups behind the slots'
__global__ __launch_bounds__(256) void pages_slots_kernel(ExtendArgs e, uint32_t slot_blocks)
{
    const PagesArgs &a = e.p;
    if (blockIdx.x < slot_blocks) {
        const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
        if (row >= e.rows)
            return;
        int slot = -1;
        if (row < e.starts[a.seqs]) {
            const int s = sequence_of(e.starts, a.seqs, row);
            if (e.granted[s] > 0)
                slot = slot_of(a, s, a.lengths[s] - e.granted[s] + (int)(row - e.starts[s]));
        }
        e.slots[row] = slot;
        return;
    }
    const int s = (blockIdx.x - slot_blocks) * 4 + (threadIdx.x >> 6);
    if (s < a.seqs && e.granted[s] < 0) {
        const int to = pages_of(a, a.lengths[s] - e.granted[s]);
        for (int j = pages_of(a, a.lengths[s]) + (threadIdx.x & 63); j < to; j += 64)
            release(a, s, j);
    }
}

// ---------------------------------------------------------------------------------------------------------- compact

// The moves, and the counts of the pages that they are about
__global__ __launch_bounds__(kScan) void pages_compact_kernel(PagesArgs a, int32_t *moves)
{
    __shared__ int32_t counted[kScan / 64];
    __shared__ int64_t sums[2][kScan / 64];
    int n = 0;
    for (int p = threadIdx.x; p < a.num_pages; p += kScan)
        n += a.refs[p] > 0;
    int32_t live;
    scan(n, counted, &live);
    // holes before page `live` in the high word, pages to be moved into them behind it in the low one
    int64_t found = 0;
    for (int base = 0, round = 0; base < a.num_pages; base += 4 * kScan, ++round) {
        const int p0 = base + 4 * threadIdx.x;
        int64_t mine[4], sum = 0, here;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = p0 + i;
            const bool taken = p < a.num_pages && a.refs[p] > 0;
            mine[i] = p >= a.num_pages ? 0 : p < live ? (int64_t)!taken << 32 : (int64_t)taken;
            sum += mine[i];
        }
        int64_t at = found + scan(sum, sums[round & 1], &here);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (mine[i])
                moves[mine[i] == 1 ? 2 * (int64_t)(uint32_t)at : 2 * (at >> 32) + 1] = p0 + i;
            at += mine[i];
        }
        found += here;
    }
    const int count = (int)(uint32_t)found, most = a.num_pages / 2;
    __syncthreads();
    for (int i = threadIdx.x; i < most; i += kScan) {
        if (i < count) {
            const int from = moves[2 * i], to = moves[2 * i + 1];
            a.refs[to] = a.refs[from];
            a.refs[from] = 0;
        } else
            moves[2 * i] = moves[2 * i + 1] = -1;
    }
}

__global__ __launch_bounds__(256) void pages_rename_kernel(PagesArgs a, const int32_t *moves)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.seqs * a.max_pages)
        return;
    const int32_t page = a.table[i];
    if (!is_page(a, page) || (uint32_t)page < (uint32_t)moves[0])
        return; // (without moves the first is -1, as an unsigned number beyond all pages)
    int lo = 0, hi = a.num_pages / 2;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if ((uint32_t)moves[2 * (int64_t)mid] < (uint32_t)page)
            lo = mid + 1;
        else
            hi = mid;
    }
    if (lo < a.num_pages / 2 && moves[2 * (int64_t)lo] == page)
        a.table[i] = moves[2 * (int64_t)lo + 1];
}

// ---------------------------------------------------------------------------------------------------------- copies

// A cache's arrays, each so many 16-byte words a page and so many turns of a workgroup; bounds' scales, whose pages may be of 4 bytes, by
// themselves, as the last turn's
constexpr int kArrays = 5;
struct CopyArgs {
    uint4 *at[kArrays];
    int64_t words[kArrays];
    int32_t turns[kArrays]; // up to and with this array
    float *scales;
    int heads, num_pages;
    const int32_t *pairs;
    uint32_t each; // workgroups of a pair
};

// A turn is 4 KB, a word of a lane: with four words of a lane in 16 KB, 315 pages of 132 KB took 24 us instead of 15, three of 530 KB 10
// instead of 2.5
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a)
{
    const uint32_t pair = blockIdx.x / a.each;
    const int from = a.pairs[2 * (int64_t)pair], to = a.pairs[2 * (int64_t)pair + 1];
    if ((uint32_t)from >= (uint32_t)a.num_pages || (uint32_t)to >= (uint32_t)a.num_pages || from == to)
        return;
    for (int turn = (int)(blockIdx.x % a.each); turn < a.turns[kArrays - 1]; turn += (int)a.each) {
        uint4 *at = a.at[0];
        int64_t n = a.words[0], i = turn;
#pragma unroll
        for (int k = 1; k < kArrays; ++k)
            if (turn >= a.turns[k - 1]) {
                at = a.at[k];
                n = a.words[k];
                i = turn - a.turns[k - 1];
            }
        i = i * 256 + threadIdx.x;
        if (i < n)
            at[to * n + i] = at[from * n + i];
        if (a.scales && turn == a.turns[kArrays - 1] - 1)
            for (int h = threadIdx.x; h < a.heads; h += 256)
                a.scales[(int64_t)to * a.heads + h] = a.scales[(int64_t)from * a.heads + h];
    }
}

PagesArgs pages_args(const abq_kv_pages &p)
{
    return {p.table, p.lengths, p.refs, p.seqs, p.max_pages, p.num_pages, __builtin_ctz((unsigned)p.page_size)};
}

} // namespace

hipError_t launch_pages_fork(const abq_kv_pages &p, const int32_t *parents, hipStream_t stream)
{
    // four columns a workgroup, where the 64 KB that a launch gets unasked hold them: enough workgroups for the tables of many sequences, 16 bytes a row
    const int shift = p.seqs <= 4096 ? 2 : 1, columns = 1 << shift;
    const dim3 grid((unsigned)((p.max_pages + columns - 1) / columns + 1));
    hipLaunchKernelGGL(pages_fork_kernel, grid, dim3(1024), sizeof(int32_t) * p.seqs << shift, stream, pages_args(p), parents, columns, shift);
    return hipGetLastError();
}

hipError_t launch_pages_extend(const abq_kv_pages &p, const int32_t *counts, int32_t *slots, int64_t rows, int32_t *starts, int32_t *granted, int32_t *copies,
                               hipStream_t stream)
{
    const ExtendArgs e = {pages_args(p), counts, slots, starts, granted, copies, rows};
    // one launch where the workgroup that scans has little else to do
    const int all = rows <= 4 * kScan;
    hipLaunchKernelGGL(pages_extend_kernel, dim3(1), dim3(kScan), 0, stream, e, all);
    if (!all) {
        const uint32_t slot_blocks = (uint32_t)((rows + 255) / 256);
        hipLaunchKernelGGL(pages_slots_kernel, dim3(slot_blocks + (p.seqs + 3) / 4), dim3(256), 0, stream, e, slot_blocks);
    }
    return hipGetLastError();
}

hipError_t launch_pages_compact(const abq_kv_pages &p, int32_t *moves, hipStream_t stream)
{
    if (p.num_pages < 2)
        return hipSuccess;
    const PagesArgs a = pages_args(p);
    hipLaunchKernelGGL(pages_compact_kernel, dim3(1), dim3(kScan), 0, stream, a, moves);
    hipLaunchKernelGGL(pages_rename_kernel, dim3((unsigned)(((int64_t)p.seqs * p.max_pages + 255) / 256)), dim3(256), 0, stream, a, moves);
    return hipGetLastError();
}

hipError_t launch_copy_pages(const abq_kv_cache &c, const abq_kv_bounds *bounds, const int32_t *pairs, int64_t count, hipStream_t stream)
{
    if (count == 0)
        return hipSuccess;
    CopyArgs a = {};
    const int64_t rows = (int64_t)c.page_size * c.kv_heads, codes = rows * c.head_dim * c.bits / 8 / 16, scales = rows * (c.symmetric ? 1 : 2) / 4;
    void *at[kArrays] = {c.k_codes, c.v_codes, c.k_scales, c.v_scales, bounds ? bounds->codes : nullptr};
    const int64_t words[kArrays] = {codes, codes, scales, scales, bounds ? (int64_t)c.kv_heads * 2 * c.head_dim / 16 : 0};
    for (int i = 0; i < kArrays; ++i) {
        a.at[i] = (uint4 *)at[i];
        a.words[i] = words[i];
        a.turns[i] = (i ? a.turns[i - 1] : 0) + (int)((words[i] + 255) / 256);
    }
    a.scales = bounds ? bounds->scales : nullptr;
    a.heads = c.kv_heads;
    a.num_pages = c.num_pages;
    a.pairs = pairs;
    const int64_t most = kMostBlocks / count;
    a.each = (uint32_t)(a.turns[kArrays - 1] < most ? a.turns[kArrays - 1] : most);
    hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)(count * a.each)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

} // namespace abq
