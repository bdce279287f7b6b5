// paged_cache.hip — the paged KV cache's own kernels: appending rows,
// choosing the pages that sparse attention reads, and eviction.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "device.hpp"
#include "paged_device.hpp"
#include "runtime.hpp"

namespace nut {

namespace {

// ---------------------------------------------------------------- append --

// A workgroup per (sequence, KV head, page that gains rows): it alone touches
// the page's bounds, so they need no atomics. tpr = head_dim / 8 threads hold
// a row, eight components (32 bytes of source) each.
template <int TYPE>
__global__ __launch_bounds__(256) void append_kernel(
    PagedView kv, PagedSeqs s, const float *__restrict__ keys, const float *__restrict__ values,
    size_t rows, size_t row_stride, size_t head_stride, const int *__restrict__ starts,
    uint32_t each, uint32_t max_new, PagedHistory history, const int *__restrict__ firsts, int *new_lengths,
    uint32_t touched)
{
    const uint32_t id = blockIdx.x;
    const uint32_t c = id % touched, h = id / touched % kv.kv_heads;
    const uint32_t b = id / touched / kv.kv_heads;
    const bool leader = threadIdx.x == 0 && h == 0 && c == 0;

    const int length = s.lengths[b];
    const int64_t from = starts == nullptr ? int64_t(b) * each : starts[b];
    int64_t gain = starts == nullptr ? int64_t(each) : starts[b + 1] - from;
    int bad = 0;
    if (from < 0 || gain < 0 || gain > int64_t(max_new) || from + gain > int64_t(rows))
        bad = kBadRows, gain = 0;
    else if (length < 0 || length + gain > int64_t(s.max_length))
        bad = kBadLength, gain = 0;
    if (leader) {
        if (bad != 0)
            paged_flag(kv.status, bad);
        if (new_lengths != nullptr)
            new_lengths[b] = length + int(gain);
    }
    if (gain == 0)
        return;

    const uint32_t n = uint32_t(length), m = uint32_t(gain), ps = kv.page_size;
    const uint32_t index = n / ps + c;
    // 64 bits: the end of the last page may pass 32
    const uint32_t begin = max(n, index * ps);
    const uint32_t end = uint32_t(min(uint64_t(n) + m, (uint64_t(index) + 1) * ps));
    if (uint64_t(index) * ps >= uint64_t(n) + m)
        return;
    if (history.weights != nullptr) {
        const size_t at = (size_t(b) * kv.kv_heads + h) * history.stride;
        const int first = firsts == nullptr ? length : firsts[b];
        for (uint32_t r = begin + threadIdx.x; r < end; r += blockDim.x) {
            history.weights[at + r] = 0.0f;
            history.positions[at + r] = first + int(r - n);
        }
    }
    const size_t page = paged_row(kv, s, b, index, 0, h);
    if (page == kNoRow)
        return;

    const uint32_t tpr = kv.head_dim / 8, part = threadIdx.x % tpr, group = threadIdx.x / tpr;
    const uint32_t groups = blockDim.x / tpr;
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        lo[i] = INFINITY, hi[i] = -INFINITY;
    if (group < groups)
        for (uint32_t r = begin + group; r < end; r += groups) {
            const size_t source = (size_t(from) + (r - n)) * row_stride + h * head_stride + part * 8;
            const size_t to = page + size_t(r - index * ps) * kv.slot_stride +
                              part * 8 * (TYPE == NUT_F32 ? 4 : 2);
            float k[8], v[8];
            load8<NUT_F32>(reinterpret_cast<const char *>(keys + source), k);
            load8<NUT_F32>(reinterpret_cast<const char *>(values + source), v);
            store8<TYPE>(kv.keys + to, k);
            store8<TYPE>(kv.values + to, v);
#pragma unroll
            for (int i = 0; i < 8; i++)
                lo[i] = lower(lo[i], k[i]), hi[i] = upper(hi[i], k[i]);
        }
    if (kv.bounds == nullptr)
        return;
    __shared__ float low[256][8], high[256][8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        low[threadIdx.x][i] = lo[i], high[threadIdx.x][i] = hi[i];
    __syncthreads();
    const uint32_t used = min(groups, end - begin);
    char *bounds = kv.bounds + (size_t(s.table[size_t(b) * s.table_stride + index]) * kv.kv_heads +
                                h) * 2 * kv.head_dim * (TYPE == NUT_F32 ? 4 : 2);
    for (uint32_t p = threadIdx.x; p < tpr; p += blockDim.x) {
        float a[8], z[8];
        const size_t size = TYPE == NUT_F32 ? 4 : 2;
        if (index * ps < n) {
            load8<TYPE>(bounds + p * 8 * size, a);
            load8<TYPE>(bounds + (kv.head_dim + p * 8) * size, z);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                a[i] = INFINITY, z[i] = -INFINITY;
        }
        for (uint32_t g = 0; g < used; g++)
#pragma unroll
            for (int i = 0; i < 8; i++)
                a[i] = lower(a[i], low[g * tpr + p][i]), z[i] = upper(z[i], high[g * tpr + p][i]);
        store8<TYPE>(bounds + p * 8 * size, a);
        store8<TYPE>(bounds + (kv.head_dim + p * 8) * size, z);
    }
}

// ------------------------------------------------------ the k-th largest --

constexpr int kBits = 11, kBins = 1 << kBits;

struct RankScratch {
    uint32_t bins[kBins];
    uint32_t wave[16], more[16];
    uint32_t bin, above, count;
    unsigned long long any, all;
};

// Finds, for keys get(0) to get(n - 1) and 1 <= k < n, the threshold T and
// the number of ties such that the k largest keys, ties to the lowest index,
// are the keys over T and the first `ties` keys equal to T. A radix search
// from the first bit in which the keys differ, 11 bits a pass, which ends at
// the first digit whose keys are all taken (scores differ in their leading
// bits: two or three passes). Every thread of the workgroup calls it.
template <typename K, typename Get>
__device__ __forceinline__ void kth_largest(Get get, uint32_t n, uint32_t k, RankScratch &sc,
                                            K &threshold, uint32_t &ties)
{
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const uint32_t waves = blockDim.x / kWave;
    if (threadIdx.x == 0)
        sc.any = 0, sc.all = ~0ull;
    __syncthreads();
    K any = 0, all = K(~K(0));
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const K key = get(i);
        any |= key, all &= key;
    }
    atomicOr(&sc.any, (unsigned long long)any);
    atomicAnd(&sc.all, (unsigned long long)all);
    __syncthreads();
    any = K(sc.any), all = K(sc.all);
    const K differ = any ^ all;
    if (differ == 0) {
        threshold = any;
        ties = k;
        __syncthreads();
        return;
    }
    int shift = 64 - __clzll((unsigned long long)differ); // bits still open
    K prefix = shift >= int(8 * sizeof(K)) ? K(0) : K(any >> shift << shift);
    uint32_t left = k;
    while (true) {
        const int width = min(kBits, shift), top = shift;
        shift -= width;
        for (uint32_t i = threadIdx.x; i < kBins; i += blockDim.x)
            sc.bins[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
            const K key = get(i);
            const K open = key ^ prefix;
            if (top >= int(8 * sizeof(K)) || (open >> top) == 0)
                atomicAdd(&sc.bins[uint32_t(key >> shift) & ((1u << width) - 1)], 1u);
        }
        __syncthreads();
        // thread t owns `own` bins, from the highest down
        const uint32_t own = kBins / blockDim.x, high = kBins - 1 - threadIdx.x * own;
        uint32_t sum = 0;
        for (uint32_t i = 0; i < own; i++)
            sum += sc.bins[high - i];
        uint32_t scan = sum;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const uint32_t up = __shfl_up(scan, o);
            scan += lane >= uint32_t(o) ? up : 0;
        }
        if (lane == kWave - 1)
            sc.wave[wave] = scan;
        __syncthreads();
        for (uint32_t w = 0; w < wave; w++)
            scan += sc.wave[w];
        if (scan >= left && scan - sum < left) {
            uint32_t above = scan - sum, i = 0;
            while (above + sc.bins[high - i] < left)
                above += sc.bins[high - i++];
            sc.bin = high - i, sc.above = above, sc.count = sc.bins[high - i];
        }
        __syncthreads();
        prefix |= K(sc.bin) << shift;
        left -= sc.above;
        const bool whole = sc.count == left;
        __syncthreads();
        if (whole || shift == 0) {
            threshold = prefix;
            ties = whole ? 0xffffffffu : left;
            return;
        }
    }
    (void)waves;
}

// Lanes below this one in a ballot.
__device__ __forceinline__ uint32_t rank_in(uint64_t mask)
{
    return __builtin_amdgcn_mbcnt_hi(uint32_t(mask >> 32),
                                     __builtin_amdgcn_mbcnt_lo(uint32_t(mask), 0));
}

// ---------------------------------------------------------------- select --

// Order-preserving image of a score; a NaN ranks above every number, the
// pages that are always read above both.
__device__ __forceinline__ uint64_t score_key(double v)
{
    if (v != v)
        return ~0ull - 1;
    const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0); // -0 ranks as 0
    return u >> 63 ? ~u : u | (1ull << 63);
}

// Scores of every page: `lanes` lanes (a power of two, head_dim / 8 of them
// with work) hold eight components of a page's bounds each. For one page
//   sum_d max(q_d lo_d, q_d hi_d) = sum_d q_d (hi_d + lo_d) / 2
//                                        + |q_d| (hi_d - lo_d) / 2,
// two multiply-adds a component in 64 bits: the answer is whole numbers, and
// 32 bits would let rounding choose among near pages. GH heads at a time.
template <int TYPE, int GH>
__global__ __launch_bounds__(256) void page_scores_kernel(PagedView kv, PagedSeqs s,
                                                          const float *__restrict__ query,
                                                          size_t query_stride, uint32_t heads,
                                                          uint32_t lanes, uint32_t per_block,
                                                          uint32_t blocks, uint32_t width,
                                                          uint64_t *__restrict__ scores)
{
    const uint32_t id = blockIdx.x, c = id % blocks, h = id / blocks % kv.kv_heads;
    const uint32_t b = id / blocks / kv.kv_heads;
    const uint32_t n = paged_length(kv, s, b, threadIdx.x == 0 && h == 0 && c == 0);
    const uint32_t count = n / kv.page_size + (n % kv.page_size != 0);
    if (c * per_block >= count)
        return;
    const uint32_t end = min(count, (c + 1) * per_block);
    const uint32_t group = heads / kv.kv_heads, part = threadIdx.x % lanes;
    const size_t size = TYPE == NUT_F32 ? 4 : 2;
    const bool works = part * 8 < kv.head_dim;
    uint64_t *out = scores + (size_t(b) * kv.kv_heads + h) * width;
    for (uint32_t g = 0; g < group; g += GH) {
        double q[GH][8];
#pragma unroll
        for (int j = 0; j < GH; j++) {
            float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (works && g + j < group)
                load8<NUT_F32>(reinterpret_cast<const char *>(
                                   query + b * query_stride +
                                   size_t(h * group + g + j) * kv.head_dim + part * 8),
                               v);
#pragma unroll
            for (int i = 0; i < 8; i++)
                q[j][i] = double(v[i]);
        }
        for (uint32_t p = c * per_block + threadIdx.x / lanes; p < end; p += 256 / lanes) {
            const int page = s.table[size_t(b) * s.table_stride + p];
            const bool good = page >= 0 && uint32_t(page) < kv.pages;
            if (!good && part == 0)
                paged_flag(kv.status, kBadPage);
            double mid[8], half[8];
            {
                float lo[8] = {0, 0, 0, 0, 0, 0, 0, 0}, hi[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (good && works) {
                    const char *at = kv.bounds + (size_t(page) * kv.kv_heads + h) * 2 *
                                                     kv.head_dim * size + part * 8 * size;
                    load8<TYPE>(at, lo);
                    load8<TYPE>(at + kv.head_dim * size, hi);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    mid[i] = 0.5 * (double(hi[i]) + double(lo[i]));
                    half[i] = 0.5 * (double(hi[i]) - double(lo[i]));
                }
            }
            uint64_t best = 0;
#pragma unroll
            for (int j = 0; j < GH; j++) {
                double sum = 0.0;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    sum = fma(fabs(q[j][i]), half[i], fma(q[j][i], mid[i], sum));
                for (uint32_t o = 1; o < lanes; o <<= 1)
                    sum += __shfl_xor(sum, int(o));
                const uint64_t key = score_key(sum);
                if (g + j < group && key > best)
                    best = key;
            }
            if (part == 0) {
                if (!good)
                    best = 0;
                out[p] = g == 0 ? best : (best > out[p] ? best : out[p]);
            }
        }
    }
}

// A workgroup per (sequence, KV head): the `top` best of its pages.
__global__ __launch_bounds__(256) void choose_pages_kernel(PagedView kv, PagedSeqs s,
                                                           const uint64_t *__restrict__ scores,
                                                           uint32_t width, uint32_t top,
                                                           uint32_t first, uint32_t last,
                                                           int *__restrict__ selected)
{
    const uint32_t id = blockIdx.x, h = id % kv.kv_heads, b = id / kv.kv_heads;
    const uint32_t n = paged_length(kv, s, b, false);
    const uint32_t count = n / kv.page_size + (n % kv.page_size != 0);
    int *out = selected + (size_t(b) * kv.kv_heads + h) * top;
    if (count <= top) {
        for (uint32_t i = threadIdx.x; i < top; i += blockDim.x)
            out[i] = i < count ? int(i) : -1;
        return;
    }
    __shared__ RankScratch sc;
    const uint64_t *mine = scores + (size_t(b) * kv.kv_heads + h) * width;
    const auto get = [&](uint32_t i) -> uint64_t {
        return i < first || i >= count - last ? ~0ull : mine[i];
    };
    uint64_t threshold;
    uint32_t ties;
    kth_largest<uint64_t>(get, count, top, sc, threshold, ties);

    // each wave writes what is kept of a run of pages of its own
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const uint32_t run = (count + blockDim.x - 1) / blockDim.x * kWave;
    const uint32_t begin = min(count, wave * run), end = min(count, begin + run);
    uint32_t over = 0, equal = 0;
    for (uint32_t i = begin + lane; i < end; i += kWave) {
        const uint64_t key = get(i);
        over += key > threshold, equal += key == threshold;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        over += __shfl_xor(over, o), equal += __shfl_xor(equal, o);
    if (lane == 0)
        sc.wave[wave] = over, sc.more[wave] = equal;
    __syncthreads();
    uint32_t at = 0, seen = 0;
    for (uint32_t w = 0; w < wave; w++)
        at += sc.wave[w], seen += sc.more[w];
    at += min(seen, ties);
    for (uint32_t base = begin; base < end; base += kWave) {
        const uint32_t i = base + lane;
        const uint64_t key = i < end ? get(i) : 0;
        const bool tie = i < end && key == threshold;
        const uint64_t tied = __ballot(tie);
        const bool kept = i < end && (key > threshold || (tie && seen + rank_in(tied) < ties));
        const uint64_t all = __ballot(kept);
        if (kept)
            out[at + rank_in(all)] = int(i);
        at += __popcll(all);
        seen += __popcll(tied);
    }
}

// ----------------------------------------------------------------- evict --

__device__ __forceinline__ uint32_t weight_key(float w)
{
    if (w != w)
        return 0;
    const uint32_t u = __float_as_uint(w + 0.0f);
    const uint32_t key = u >> 31 ? ~u : u | 0x80000000u;
    return key; // at least ~0xff800000 = 0x007fffff, over a NaN's
}

// A workgroup per (sequence, KV head) decides what stays: moves[i] of a row
// i below the budget is -1 where it stays and its rank among the holes where
// it goes; from[r] is the r-th row that stays beyond the budget.
__global__ __launch_bounds__(1024) void plan_eviction_kernel(PagedView kv, PagedSeqs s,
                                                             PagedHistory history,
                                                             uint32_t budget, uint32_t first,
                                                             uint32_t last, int *new_lengths,
                                                             int *__restrict__ moves,
                                                             int *__restrict__ from)
{
    const uint32_t id = blockIdx.x, h = id % kv.kv_heads, b = id / kv.kv_heads;
    const bool leader = threadIdx.x == 0 && h == 0;
    const uint32_t n = paged_length(kv, s, b, leader);
    if (leader) {
        const int was = s.lengths[b];
        new_lengths[b] = n > budget ? int(budget) : was;
    }
    if (n <= budget)
        return;
    __shared__ RankScratch sc;
    __shared__ int newest_of[16];
    const size_t at = (size_t(b) * kv.kv_heads + h) * history.stride;
    const float *weights = history.weights + at;
    const int *positions = history.positions + at;
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    int newest = -1;
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x)
        newest = max(newest, positions[i]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        newest = max(newest, __shfl_xor(newest, o));
    if (lane == 0)
        newest_of[wave] = newest;
    __syncthreads();
    for (uint32_t w = 0; w < blockDim.x / kWave; w++)
        newest = max(newest, newest_of[w]);
    const int64_t recent = int64_t(newest) - int64_t(last);
    const auto get = [&](uint32_t i) -> uint32_t {
        const int p = positions[i];
        return p < int64_t(first) || p > recent ? 0xffffffffu : weight_key(weights[i]);
    };
    uint32_t threshold, ties;
    kth_largest<uint32_t>(get, n, budget, sc, threshold, ties);

    const uint32_t run = (n + blockDim.x - 1) / blockDim.x * kWave;
    const uint32_t begin = min(n, wave * run), end = min(n, begin + run);
    uint32_t equal = 0;
    for (uint32_t i = begin + lane; i < end; i += kWave)
        equal += get(i) == threshold;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        equal += __shfl_xor(equal, o);
    if (lane == 0)
        sc.more[wave] = equal;
    __syncthreads();
    uint32_t seen = 0;
    for (uint32_t w = 0; w < wave; w++)
        seen += sc.more[w];
    // walk the run twice: count its holes and its rows to move, then place them
    uint32_t holes = 0, moved = 0;
    int *move = moves + (size_t(b) * kv.kv_heads + h) * budget;
    int *source = from + (size_t(b) * kv.kv_heads + h) * budget;
    for (int pass = 0; pass < 2; pass++) {
        uint32_t met = seen;
        for (uint32_t base = begin; base < end; base += kWave) {
            const uint32_t i = base + lane;
            const uint32_t key = i < end ? get(i) : 0;
            const bool tie = i < end && key == threshold;
            const uint64_t tied = __ballot(tie);
            const bool kept = i < end && (key > threshold || (tie && met + rank_in(tied) < ties));
            const uint64_t hole = __ballot(i < end && i < budget && !kept);
            const uint64_t goes = __ballot(kept && i >= budget);
            if (pass == 1) {
                if (i < end && i < budget)
                    move[i] = kept ? -1 : int(holes + rank_in(hole));
                else if (kept)
                    source[moved + rank_in(goes)] = int(i);
            }
            holes += __popcll(hole);
            moved += __popcll(goes);
            met += __popcll(tied);
        }
        if (pass == 0) {
            if (lane == 0)
                sc.wave[wave] = holes, sc.bins[wave] = moved;
            __syncthreads();
            holes = moved = 0;
            for (uint32_t w = 0; w < wave; w++)
                holes += sc.wave[w], moved += sc.bins[w];
        }
    }
}

// A workgroup per (sequence, KV head, page below the budget) fetches what
// moves into the page. Sources lie beyond the budget and are only read, so
// the order of workgroups does not matter.
template <int TYPE>
__global__ __launch_bounds__(256) void move_rows_kernel(PagedView kv, PagedSeqs s,
                                                        PagedHistory history, uint32_t budget,
                                                        uint32_t pages,
                                                        const int *__restrict__ moves,
                                                        const int *__restrict__ from)
{
    const uint32_t id = blockIdx.x, c = id % pages, h = id / pages % kv.kv_heads;
    const uint32_t b = id / pages / kv.kv_heads;
    const uint32_t n = paged_length(kv, s, b, false);
    if (n <= budget)
        return;
    const uint32_t ps = kv.page_size, first = c * ps, end = min(budget - first, ps);
    const size_t row = size_t(b) * kv.kv_heads + h, at = row * history.stride;
    const int *move = moves + row * budget + first, *source = from + row * budget;
    const size_t page = paged_row(kv, s, b, c, 0, h);
    const uint32_t tpr = kv.head_dim / 8, part = threadIdx.x % tpr, group = threadIdx.x / tpr;
    const uint32_t groups = 256 / tpr;
    const size_t size = TYPE == NUT_F32 ? 4 : 2, column = part * 8 * size;
    __shared__ int sources[256];
    __shared__ float low[256][8], high[256][8];
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        lo[i] = INFINITY, hi[i] = -INFINITY;
    bool some = false;
    for (uint32_t w = 0; w < end; w += 256) {
        const uint32_t slot = w + threadIdx.x;
        const int rank = slot < end ? move[slot] : -1;
        const int src = rank < 0 ? -1 : source[rank];
        if (src >= 0) {
            history.weights[at + first + slot] = history.weights[at + src];
            history.positions[at + first + slot] = history.positions[at + src];
        }
        sources[threadIdx.x] = src;
        if (__syncthreads_or(src >= 0) && page != kNoRow && group < groups) {
            for (uint32_t r = group; r < min(end - w, 256u); r += groups) {
                const int i = sources[r];
                if (i < 0)
                    continue;
                const size_t there = paged_row(kv, s, b, uint32_t(i) / ps, uint32_t(i) % ps, h);
                if (there == kNoRow)
                    continue;
                some = true;
                const size_t here = page + size_t(w + r) * kv.slot_stride + column;
                const uint4 *k = reinterpret_cast<const uint4 *>(kv.keys + there + column);
                const uint4 *v = reinterpret_cast<const uint4 *>(kv.values + there + column);
                uint4 *to_k = reinterpret_cast<uint4 *>(kv.keys + here);
                uint4 *to_v = reinterpret_cast<uint4 *>(kv.values + here);
                float x[8];
                load8<TYPE>(kv.keys + there + column, x);
#pragma unroll
                for (int j = 0; j < int(size / 2); j++)
                    to_k[j] = k[j], to_v[j] = v[j];
#pragma unroll
                for (int j = 0; j < 8; j++)
                    lo[j] = lower(lo[j], x[j]), hi[j] = upper(hi[j], x[j]);
            }
        }
        __syncthreads();
    }
    if (kv.bounds == nullptr || !__syncthreads_or(some))
        return;
#pragma unroll
    for (int i = 0; i < 8; i++)
        low[threadIdx.x][i] = lo[i], high[threadIdx.x][i] = hi[i];
    __syncthreads();
    if (threadIdx.x < tpr) {
        char *bounds = kv.bounds + (size_t(s.table[size_t(b) * s.table_stride + c]) *
                                        kv.kv_heads + h) * 2 * kv.head_dim * size;
        float a[8], z[8];
        load8<TYPE>(bounds + column, a);
        load8<TYPE>(bounds + kv.head_dim * size + column, z);
        for (uint32_t g = 0; g < groups; g++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                a[i] = lower(a[i], low[g * tpr + part][i]);
                z[i] = upper(z[i], high[g * tpr + part][i]);
            }
        store8<TYPE>(bounds + column, a);
        store8<TYPE>(bounds + kv.head_dim * size + column, z);
    }
}

uint32_t pages_of(const PagedView &kv, uint32_t rows) { return (rows - 1) / kv.page_size + 1; }

size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

template <int TYPE>
void scores_for(const PagedView &kv, const PagedSeqs &seqs, const float *query,
                size_t query_stride, uint32_t heads, uint64_t *scores, hipStream_t stream)
{
    uint32_t lanes = 1;
    while (lanes * 8 < kv.head_dim)
        lanes *= 2;
    const uint32_t width = pages_of(kv, seqs.max_length), group = heads / kv.kv_heads;
    const uint32_t per_block = 256 / lanes * 4, blocks = (width + per_block - 1) / per_block;
    const dim3 grid = paged_grid(uint64_t(seqs.batch) * kv.kv_heads * blocks, 256);
    const auto kernel = group == 1   ? page_scores_kernel<TYPE, 1>
                        : group == 2 ? page_scores_kernel<TYPE, 2>
                        : group <= 4 ? page_scores_kernel<TYPE, 4>
                                     : page_scores_kernel<TYPE, 8>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, kv, seqs, query, query_stride, heads,
                       lanes, per_block, blocks, width, scores);
}

} // namespace

void launch_paged_append(const PagedView &kv, const PagedSeqs &seqs, const float *keys,
                         const float *values, size_t rows, size_t row_stride,
                         size_t head_stride, const int *starts, uint32_t each,
                         uint32_t max_new, const PagedHistory &history, const int *firsts,
                         int *new_lengths, hipStream_t stream)
{
    // pages that max_new rows can lie in, wherever they begin
    const uint32_t touched = (max_new - 1 + kv.page_size - 1) / kv.page_size + 1;
    const uint32_t most = std::min(kv.page_size, max_new) * (kv.head_dim / 8);
    const uint32_t threads = std::min(256u, (most + kWave - 1) / kWave * kWave);
    const auto kernel = kv.type == NUT_F32   ? append_kernel<NUT_F32>
                        : kv.type == NUT_F16 ? append_kernel<NUT_F16>
                                             : append_kernel<NUT_BF16>;
    hipLaunchKernelGGL(kernel, paged_grid(uint64_t(seqs.batch) * kv.kv_heads * touched, threads),
                       dim3(threads), 0, stream, kv, seqs, keys, values, rows, row_stride, head_stride, starts, each,
                       max_new, history, firsts, new_lengths, touched);
    check_launch("paged append");
}

size_t select_workspace(const PagedView &kv, const PagedSeqs &seqs)
{
    return size_t(seqs.batch) * kv.kv_heads * pages_of(kv, seqs.max_length) * sizeof(uint64_t);
}

void launch_paged_select(const PagedView &kv, const PagedSeqs &seqs, const float *query,
                         size_t query_stride, uint32_t heads, uint32_t top, uint32_t first,
                         uint32_t last, int *selected, char *workspace, hipStream_t stream)
{
    uint64_t *scores = reinterpret_cast<uint64_t *>(workspace);
    const auto run = kv.type == NUT_F32   ? scores_for<NUT_F32>
                     : kv.type == NUT_F16 ? scores_for<NUT_F16>
                                          : scores_for<NUT_BF16>;
    run(kv, seqs, query, query_stride, heads, scores, stream);
    check_launch("paged select");
    hipLaunchKernelGGL(choose_pages_kernel, paged_grid(uint64_t(seqs.batch) * kv.kv_heads, 256),
                       dim3(256), 0, stream, kv, seqs, scores, pages_of(kv, seqs.max_length), top, first, last,
                       selected);
    check_launch("paged select");
}

size_t evict_workspace(const PagedView &kv, const PagedSeqs &seqs, uint32_t budget)
{
    return 2 * aligned(size_t(seqs.batch) * kv.kv_heads * budget * sizeof(int));
}

void launch_paged_evict(const PagedView &kv, const PagedSeqs &seqs, const PagedHistory &history,
                        uint32_t budget, uint32_t first, uint32_t last, int *new_lengths,
                        char *workspace, hipStream_t stream)
{
    int *moves = reinterpret_cast<int *>(workspace);
    int *from = reinterpret_cast<int *>(workspace + evict_workspace(kv, seqs, budget) / 2);
    const uint64_t heads = uint64_t(seqs.batch) * kv.kv_heads;
    hipLaunchKernelGGL(plan_eviction_kernel, paged_grid(heads, 1024), dim3(1024), 0, stream, kv, seqs, history,
                       budget, first, last, new_lengths, moves, from);
    check_launch("paged evict");
    if (budget >= seqs.max_length)
        return;
    const uint32_t pages = pages_of(kv, budget);
    const auto kernel = kv.type == NUT_F32   ? move_rows_kernel<NUT_F32>
                        : kv.type == NUT_F16 ? move_rows_kernel<NUT_F16>
                                             : move_rows_kernel<NUT_BF16>;
    hipLaunchKernelGGL(kernel, paged_grid(heads * pages, 256), dim3(256), 0, stream, kv, seqs, history,
                       budget, pages, moves, from);
    check_launch("paged evict");
}

} // namespace nut
