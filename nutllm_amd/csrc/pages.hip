// pages.hip — page pools of the paged KV cache: tables that go from one step to
// the next, moves out of a cache's upper part, and the copies that both ask for.
//
// A page is free where its count of references is 0, so that there is no list of
// free pages to keep: a workgroup per segment of the counts lists the free pages
// of the segment in order, and the r-th free page of all is found by the
// segments' counts.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "device.hpp"
#include "paged_device.hpp"
#include "runtime.hpp"
#include "serving.hpp"

namespace nut {

namespace {

constexpr uint32_t kSegments = 256;     // at most
constexpr uint32_t kSpan = 4096;        // pages that a workgroup lists at once
constexpr uint32_t kPlanThreads = 1024;
constexpr uint32_t kFew = 16384; // entries of a table, and copies, that one workgroup follows
constexpr uint32_t kFewHeld = 128; // and sequences
constexpr uint32_t kCounted = 2048;     // old sequences that shared memory counts
constexpr int kNone = 0x7fffffff;

// Pages of a segment, a multiple of kSpan.
uint32_t segment_of(uint32_t pages)
{
    const uint64_t each = (uint64_t(pages) + kSegments - 1) / kSegments;
    return uint32_t((each + kSpan - 1) / kSpan * kSpan);
}

__device__ __forceinline__ uint32_t wave_prefix(uint32_t v) // with this lane's
{
    const uint32_t lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const uint32_t x = __shfl_up(v, o);
        v += lane >= uint32_t(o) ? x : 0;
    }
    return v;
}

// Sum of the values of the threads before this one; `total` of all of them.
// `scratch` holds a word per wave.
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t *scratch, uint32_t &total)
{
    const uint32_t wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
    const uint32_t sum = wave_prefix(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == kWave - 1)
        scratch[wave] = sum;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
    for (uint32_t w = 0; w < waves; w++) {
        before += w < wave ? scratch[w] : 0;
        total += scratch[w];
    }
    return before + sum - v;
}

// Lists the pages of [begin, end) that `takes` in ascending order from
// list[begin] on; returns how many, in every thread.
template <int THREADS, typename Takes>
__device__ __forceinline__ uint32_t list_pages(uint32_t begin, uint32_t end, int *list,
                                               Takes &&takes)
{
    constexpr int kEach = kSpan / THREADS, kWaves = THREADS / kWave;
    __shared__ uint32_t counts[kEach * kWaves];
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    uint32_t listed = 0;
    for (uint32_t at = begin; at < end; at += kSpan) {
        uint64_t found[kEach];
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            const uint32_t p = at + e * THREADS + threadIdx.x;
            found[e] = __ballot(p < end && takes(p));
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kEach; e++)
            if (lane == 0)
                counts[e * kWaves + wave] = uint32_t(__popcll(found[e]));
        __syncthreads();
        static_assert(kEach * kWaves == kWave, "a lane a count");
        const uint32_t mine = counts[lane], upto = wave_prefix(mine);
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            const int slot = e * kWaves + wave;
            const uint32_t first = listed + __shfl(upto - mine, slot);
            if (found[e] >> lane & 1)
                list[begin + first + __popcll(found[e] & ((uint64_t(1) << lane) - 1))] =
                    int(at + e * THREADS + threadIdx.x);
        }
        listed += __shfl(upto, kWave - 1);
    }
    return listed;
}

// The segments' counts, summed: sums[i] of those before segment i. A wave's work,
// kSegments + 1 words; returns the sum of all.
__device__ __forceinline__ uint32_t sum_segments(const uint32_t *counts, uint32_t segments,
                                                 uint32_t *sums)
{
    const uint32_t lane = threadIdx.x & (kWave - 1);
    uint32_t all = 0;
    for (uint32_t at = 0; at < segments; at += kWave) {
        const uint32_t mine = at + lane < segments ? counts[at + lane] : 0;
        const uint32_t upto = wave_prefix(mine);
        sums[at + lane] = all + upto - mine; // kSegments is a multiple of kWave
        all += __shfl(upto, kWave - 1);
    }
    return all;
}

// The page of rank r, below the sum of all.
__device__ __forceinline__ int ranked_page(const int *list, const uint32_t *sums,
                                           uint32_t segments, uint32_t segment, uint32_t r)
{
    uint32_t lo = 0, hi = segments; // sums[lo] <= r, and of the last such one
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (sums[mid] <= r)
            lo = mid;
        else
            hi = mid;
    }
    return list[size_t(lo) * segment + (r - sums[lo])];
}

// --------------------------------------------------------------- reorder --

// A sequence of the new table: entries below `full` are the parent's, those up
// to `need` its own, the fresh ones of them ranks `base` onwards. parent -1: none.
struct Step {
    int parent;
    uint32_t full, need, base;
};

struct ReorderArgs {
    PoolView pool;
    TableView from, to;
    PageDivision division;
    const int *parents, *gains;
    uint32_t gain;
    int *copies;
    int *children, *first; // [from.batch]
    Step *steps;           // [to.batch]
    uint32_t *counts;      // of the segments' free pages
    int *list;             // [pages]
    uint32_t segments, segment;
};

// Whether sequence p of the old table holds as many pages as its rows need.
__device__ __forceinline__ bool whole(const ReorderArgs &a, int length, int held)
{
    return held >= 0 && uint32_t(held) <= a.from.stride && length >= 0 &&
           uint64_t(uint32_t(held)) * a.pool.page_size >= uint32_t(length);
}

__device__ __forceinline__ int atomic_read(const int *p)
{
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Which sequences go on where, and what they need: workgroup 0. 128 sequences 3.6 us, the
// launch and four reads one after another. Entries behind
// the shared ones get the page that stays, or -2 - k for the k-th fresh one.
__device__ __forceinline__ void plan_steps(const ReorderArgs &a)
{
    __shared__ uint32_t scratch[kPlanThreads / kWave];
    // Of up to kCounted old sequences in shared memory: 3 us less than by atomics on
    // global memory, with their fences.
    __shared__ int counts[kCounted], firsts[kCounted];
    const bool small = a.from.batch <= kCounted;
    int *children = small ? counts : a.children, *first_of = small ? firsts : a.first;
    const int next = threadIdx.x < a.to.batch ? a.parents[threadIdx.x] : -1;
    for (uint32_t p = threadIdx.x; p < a.from.batch; p += blockDim.x) {
        __hip_atomic_store(&children[p], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(&first_of[p], kNone, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (!small)
        __threadfence();
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.to.batch; i += blockDim.x) {
        const int p = i == threadIdx.x ? next : a.parents[i];
        if (p >= 0 && uint32_t(p) < a.from.batch) {
            atomicAdd(&children[p], 1);
            atomicMin(&first_of[p], int(i));
        }
    }
    if (!small)
        __threadfence();
    __syncthreads();
    if (small)
        for (uint32_t p = threadIdx.x; p < a.from.batch; p += blockDim.x)
            a.children[p] = counts[p], a.first[p] = firsts[p];
    const uint32_t ps = a.pool.page_size;
    uint32_t taken = 0;
    for (uint32_t base = 0; base < a.to.batch; base += blockDim.x) {
        const uint32_t i = base + threadIdx.x;
        uint32_t fresh = 0;
        Step step{-1, 0, 0, 0};
        if (i < a.to.batch) {
            const int p = i == threadIdx.x ? next : a.parents[i];
            int bad = 0, length = 0, held = 0;
            int gain = a.gains == nullptr ? int(a.gain) : a.gains[i];
            bool first = false;
            if (p < -1 || (p >= 0 && uint32_t(p) >= a.from.batch)) {
                bad = kBadParent;
            } else if (p >= 0) {
                length = a.from.lengths[p], held = a.from.held[p];
                if (!whole(a, length, held))
                    bad = kBadLength;
                first = atomic_read(&first_of[p]) == int(i);
            }
            const uint64_t room = uint64_t(a.to.stride) * ps;
            if (bad == 0 && uint32_t(length) > room)
                bad = kBadLength;
            if (bad == 0 && (gain < 0 || uint64_t(uint32_t(length)) + uint32_t(gain) > room ||
                             uint64_t(uint32_t(length)) + uint32_t(gain) > 0x7fffffff)) {
                status_flag(a.pool.status, kBadRows);
                gain = 0;
            }
            if (bad != 0) {
                status_flag(a.pool.status, bad);
                length = 0;
            } else {
                step.parent = p;
                step.full = divide(a.division, uint32_t(length));
                const uint32_t rows = uint32_t(length) + uint32_t(gain);
                step.need = rows == 0 ? 0 : divide(a.division, rows - 1) + 1;
            }
            int *entries = a.to.pages + size_t(i) * a.to.stride;
            for (uint32_t c = step.full; c < step.need; c++) {
                int page = -1;
                if (first && c < uint32_t(held)) {
                    page = a.from.pages[size_t(p) * a.from.stride + c];
                    if (!page_in(page, a.pool.pages) || a.pool.refs[page] != 1)
                        page = -1;
                }
                entries[c] = page >= 0 ? page : -2 - int(fresh++);
            }
            a.to.lengths[i] = length;
            a.to.held[i] = int(step.need);
        }
        uint32_t all;
        step.base = taken + block_prefix(fresh, scratch, all);
        taken += all;
        if (i < a.to.batch)
            a.steps[i] = step;
    }
}

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(ReorderArgs a)
{
    if (blockIdx.x == 0) {
        plan_steps(a);
        return;
    }
    const uint32_t id = blockIdx.x - 1;
    const uint64_t begin = uint64_t(id) * a.segment;
    const uint32_t end = uint32_t(min(begin + a.segment, uint64_t(a.pool.pages)));
    const uint32_t count = list_pages<kPlanThreads>(
        uint32_t(begin), end, a.list, [&](uint32_t p) { return a.pool.refs[p] == 0; });
    if (threadIdx.x == 0)
        a.counts[id] = count;
}

// The new table's entries and copies: a wave a sequence. 128 sequences of up to 94 pages
// 4.3 us (2.6 at least), of which the table is a tenth: steps, entries and lists one after another.
__device__ __forceinline__ void fill_entries(const ReorderArgs &a, uint32_t i, uint32_t *sums)
{
    const Step step = a.steps[i];
    int *entries = a.to.pages + size_t(i) * a.to.stride;
    const int *old = a.from.pages + (step.parent < 0 ? 0 : size_t(step.parent) * a.from.stride);
    for (uint32_t c = threadIdx.x; c < step.full; c += kWave) {
        int page = old[c];
        if (!page_in(page, a.pool.pages)) {
            if (page != -1) // -1: none was free for it
                status_flag(a.pool.status, kBadPage);
            page = -1;
        }
        entries[c] = page;
    }
    const int rows = step.parent < 0 ? 0
                                     : int(uint32_t(a.to.lengths[i]) -
                                           step.full * a.pool.page_size);
    uint32_t free = ~0u; // not counted yet
    int copy[3] = {-1, -1, -1};
    for (uint32_t base = step.full; base < step.need; base += kWave) {
        const uint32_t c = base + threadIdx.x;
        int page = c < step.need ? entries[c] : 0;
        if (__any(page <= -2) && free == ~0u) {
            free = sum_segments(a.counts, a.segments, sums);
            __syncthreads();
        }
        if (page > -2)
            continue;
        const uint32_t rank = step.base + uint32_t(-2 - page);
        page = -1;
        if (rank < free) {
            page = ranked_page(a.list, sums, a.segments, a.segment, rank);
            a.pool.refs[page] = 1;
        } else {
            status_flag(a.pool.status, kNoPages);
        }
        entries[c] = page;
        if (c == step.full && rows > 0 && page >= 0) {
            const int source = old[c];
            if (page_in(source, a.pool.pages))
                copy[0] = source, copy[1] = page, copy[2] = rows;
            else if (source != -1)
                status_flag(a.pool.status, kBadPage);
        }
    }
    if (threadIdx.x == 0) // it has entry `full`
        for (int e = 0; e < 3; e++)
            a.copies[size_t(i) * 3 + e] = copy[e];
}

// What an old sequence held: its full pages are held once for each that goes on
// with it, the others by the first one where they stayed.
__device__ __forceinline__ void settle(const ReorderArgs &a, uint32_t p)
{
    const int length = a.from.lengths[p], held = a.from.held[p];
    if (held < 0 || uint32_t(held) > a.from.stride) {
        if (threadIdx.x == 0)
            status_flag(a.pool.status, kBadLength);
        return;
    }
    int children = a.children[p];
    const int first = a.first[p];
    Step step{-1, 0, 0, 0};
    // no one goes on with what does not hold its rows, or is too long for the table
    if (children == 0 || !whole(a, length, held) || a.steps[first].parent != int(p))
        children = 0;
    else
        step = a.steps[first];
    const int *old = a.from.pages + size_t(p) * a.from.stride;
    for (uint32_t c = threadIdx.x; c < uint32_t(held); c += kWave) {
        const bool shared = children != 0 && c < step.full;
        if (shared && children == 1)
            continue;
        const int page = old[c];
        if (!page_in(page, a.pool.pages)) {
            if (page != -1)
                status_flag(a.pool.status, kBadPage);
            continue;
        }
        // replaced entries never hold this page, before or after they are filled
        if (!shared && children != 0 && c < step.need &&
            a.to.pages[size_t(first) * a.to.stride + c] == page)
            continue;
        atomicAdd(&a.pool.refs[page], shared ? children - 1 : -1);
    }
}

__global__ __launch_bounds__(kWave) void fill_kernel(ReorderArgs a)
{
    __shared__ uint32_t sums[kSegments];
    if (blockIdx.x < a.to.batch)
        fill_entries(a, blockIdx.x, sums);
    else
        settle(a, blockIdx.x - a.to.batch);
}

// --------------------------------------------------------------- compact --

struct CompactArgs {
    PoolView pool;
    TableView table;
    uint32_t limit;
    int *copies;
    uint32_t count;                    // of copies
    int *held;                         // [pages]: entries of the table that name a page
    uint32_t *low_counts, *high_counts; // of the segments
    int *low, *high;                   // lists of free pages below the limit, of pages to move
    int *rank;                         // [pages]: a moving page's place in its segment
    uint32_t segments, segment;
};

__global__ void clear_kernel(CompactArgs a)
{
    const uint32_t stride = gridDim.x * blockDim.x;
    for (uint64_t p = blockIdx.x * blockDim.x + threadIdx.x; p < a.pool.pages; p += stride)
        a.held[p] = 0;
    for (uint64_t i = blockIdx.x * blockDim.x + threadIdx.x; i < uint64_t(a.count) * 3; i += stride)
        a.copies[i] = -1;
}

// Entries of sequence b; none, reported, where the table has no room for them.
__device__ __forceinline__ uint32_t held_by(const CompactArgs &a, uint32_t b, bool report)
{
    const int held = a.table.held[b];
    if (held >= 0 && uint32_t(held) <= a.table.stride)
        return uint32_t(held);
    if (report)
        status_flag(a.pool.status, kBadLength);
    return 0;
}

__global__ void count_kernel(CompactArgs a)
{
    const uint32_t b = blockIdx.x, held = held_by(a, b, threadIdx.x == 0);
    for (uint32_t c = threadIdx.x; c < held; c += blockDim.x) {
        const int page = a.table.pages[size_t(b) * a.table.stride + c];
        if (page_in(page, a.pool.pages))
            atomicAdd(&a.held[page], 1);
        else if (page != -1)
            status_flag(a.pool.status, kBadPage);
    }
}

__device__ __forceinline__ bool moving(const CompactArgs &a, uint32_t p)
{
    return p >= a.limit && a.held[p] > 0 && a.pool.refs[p] == a.held[p];
}

__global__ __launch_bounds__(kPlanThreads) void sort_kernel(CompactArgs a)
{
    const uint64_t first = uint64_t(blockIdx.x) * a.segment;
    const uint32_t begin = uint32_t(first);
    const uint32_t end = uint32_t(min(first + a.segment, uint64_t(a.pool.pages)));
    const uint32_t low = list_pages<kPlanThreads>(begin, end, a.low, [&](uint32_t p) {
        return p < a.limit && a.pool.refs[p] == 0;
    });
    __syncthreads();
    const uint32_t high = list_pages<kPlanThreads>(
        begin, end, a.high, [&](uint32_t p) { return moving(a, p); });
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < high; i += blockDim.x)
        a.rank[a.high[begin + i]] = int(i);
    if (threadIdx.x == 0)
        a.low_counts[blockIdx.x] = low, a.high_counts[blockIdx.x] = high;
}

// The first workgroups follow the table's entries, the others the pages that move.
// What moves was listed before: the counts of references change beside it.
__global__ __launch_bounds__(kWave) void move_kernel(CompactArgs a)
{
    __shared__ uint32_t low_sums[kSegments], high_sums[kSegments];
    const uint32_t low = sum_segments(a.low_counts, a.segments, low_sums);
    const uint32_t high = sum_segments(a.high_counts, a.segments, high_sums);
    const uint32_t moves = min(min(low, high), a.count);
    __syncthreads();
    if (blockIdx.x < a.table.batch) {
        const uint32_t b = blockIdx.x, held = held_by(a, b, false);
        int *entries = a.table.pages + size_t(b) * a.table.stride;
        for (uint32_t c = threadIdx.x; c < held; c += kWave) {
            const int page = entries[c];
            if (!page_in(page, a.pool.pages) || uint32_t(page) < a.limit)
                continue;
            const uint32_t s = uint32_t(page) / a.segment;
            const uint32_t k = uint32_t(a.rank[page]);
            if (k >= a.high_counts[s] || a.high[size_t(s) * a.segment + k] != page)
                continue; // it does not move
            const uint32_t rank = high_sums[s] + k;
            if (rank < moves)
                entries[c] = ranked_page(a.low, low_sums, a.segments, a.segment, rank);
        }
        return;
    }
    const uint32_t rank = (blockIdx.x - a.table.batch) * kWave + threadIdx.x;
    if (rank >= moves)
        return;
    const int from = ranked_page(a.high, high_sums, a.segments, a.segment, rank);
    const int to = ranked_page(a.low, low_sums, a.segments, a.segment, rank);
    a.pool.refs[to] = a.pool.refs[from];
    a.pool.refs[from] = 0;
    int *copy = a.copies + size_t(rank) * 3;
    copy[0] = from, copy[1] = to, copy[2] = int(a.pool.page_size);
}

// All of it by one workgroup, which saves three launches: pools of up to kSpan pages,
// tables of kFew entries and kFewHeld sequences. Counts and lists are in shared memory.
// Without copies, us, and by four launches: 64 pages, 3 sequences of 20 4.8 and 14.5;
// 4,096 pages, 64 of 64 7.3 and 14.5, 64 of 256 11.8 and 15.2, 128 of 256 18.9 and 15.5,
// 512 of 16 26.9 and 14.5.
__global__ __launch_bounds__(kPlanThreads) void compact_kernel(CompactArgs a)
{
    __shared__ int held[kSpan], low_list[kSpan], high_list[kSpan];
    // threads of a sequence: all, or as few as a wave where there are many
    uint32_t team = kPlanThreads;
    while (team > uint32_t(kWave) && kPlanThreads / team < a.table.batch)
        team /= 2;
    const uint32_t at = threadIdx.x / team, lane = threadIdx.x % team, teams = kPlanThreads / team;
    for (uint32_t p = threadIdx.x; p < a.pool.pages; p += kPlanThreads)
        held[p] = 0;
    for (uint32_t i = threadIdx.x; i < a.count * 3; i += kPlanThreads)
        a.copies[i] = -1;
    __syncthreads();
    for (uint32_t b = at; b < a.table.batch; b += teams) {
        const uint32_t entries = held_by(a, b, lane == 0);
        for (uint32_t c = lane; c < entries; c += team) {
            const int page = a.table.pages[size_t(b) * a.table.stride + c];
            if (page_in(page, a.pool.pages))
                atomicAdd(&held[page], 1);
            else if (page != -1)
                status_flag(a.pool.status, kBadPage);
        }
    }
    __syncthreads();
    const uint32_t low = list_pages<kPlanThreads>(0, a.pool.pages, low_list, [&](uint32_t p) {
        return p < a.limit && a.pool.refs[p] == 0;
    });
    __syncthreads();
    const uint32_t high = list_pages<kPlanThreads>(0, a.pool.pages, high_list, [&](uint32_t p) {
        return p >= a.limit && held[p] > 0 && a.pool.refs[p] == held[p];
    });
    __syncthreads();
    for (uint32_t p = threadIdx.x; p < a.pool.pages; p += kPlanThreads)
        held[p] = -1; // from here on where a page moves to
    __syncthreads();
    for (uint32_t r = threadIdx.x; r < min(min(low, high), a.count); r += kPlanThreads) {
        const int from = high_list[r], to = low_list[r];
        held[from] = to;
        a.pool.refs[to] = a.pool.refs[from];
        a.pool.refs[from] = 0;
        int *copy = a.copies + size_t(r) * 3;
        copy[0] = from, copy[1] = to, copy[2] = int(a.pool.page_size);
    }
    __syncthreads();
    for (uint32_t b = at; b < a.table.batch; b += teams) {
        const uint32_t entries = held_by(a, b, false);
        int *own = a.table.pages + size_t(b) * a.table.stride;
        for (uint32_t c = lane; c < entries; c += team) {
            const int page = own[c];
            if (page_in(page, a.pool.pages) && held[page] >= 0)
                own[c] = held[page];
        }
    }
}

// ------------------------------------------------------------------ copy --

// A workgroup per copy, KV head and layer: 59 copies of up to 64 fp16 rows, 32 KV
// heads of 128, 32 layers, 1.9 GB in 414 us (393 at least; 4.6 TB/s, near what a large
// copy reaches). Four layers a workgroup, with their loads in flight together, took 463.
// Of few rows the start of the workgroups bounds it: 128 entries, 25 of them copies of up
// to 16 rows, 4 KV heads of 64 bfloat16 components, 22 layers 10.0 us for 2 of bytes, as
// 9,064 of 11,264 workgroups read an entry without a copy.
__global__ __launch_bounds__(256) void copy_kernel(PagedLayers layers,
                                                   const int *__restrict__ copies,
                                                   uint32_t pieces, uint32_t bound_pieces)
{
    const PagedView &kv = layers.view;
    const uint32_t h = blockIdx.y, layer = blockIdx.z;
    const int from = copies[size_t(blockIdx.x) * 3], to = copies[size_t(blockIdx.x) * 3 + 1];
    const int rows = copies[size_t(blockIdx.x) * 3 + 2];
    if (from < 0)
        return;
    if (!page_in(from, kv.pages) || !page_in(to, kv.pages) || !length_in(rows, kv.page_size)) {
        if (threadIdx.x == 0 && h == 0 && layer == 0)
            status_flag(kv.status, length_in(rows, kv.page_size) ? kBadPage : kBadRows);
        return;
    }
    if (from == to)
        return;
    const size_t source = size_t(from) * kv.page_stride + h * kv.head_stride;
    const size_t target = size_t(to) * kv.page_stride + h * kv.head_stride;
    // threads by rows of `pieces`, keys and values in turn
    const uint32_t unit = threadIdx.x / pieces, units = blockDim.x / pieces / 2;
    char *pool = unit % 2 == 0 ? layers.keys[layer] : layers.values[layer];
    if (unit < 2 * units)
        for (uint32_t row = unit / 2; row < uint32_t(rows); row += units) {
            const size_t at = row * kv.slot_stride + (threadIdx.x - unit * pieces) * sizeof(uint4);
            *reinterpret_cast<uint4 *>(pool + target + at) =
                *reinterpret_cast<const uint4 *>(pool + source + at);
        }
    if (kv.bounds != nullptr)
        for (uint32_t i = threadIdx.x; i < bound_pieces; i += blockDim.x) {
            const size_t each = size_t(bound_pieces) * sizeof(uint4);
            char *bounds = layers.bounds[layer] + i * sizeof(uint4);
            *reinterpret_cast<uint4 *>(bounds + (size_t(to) * kv.kv_heads + h) * each) =
                *reinterpret_cast<const uint4 *>(bounds + (size_t(from) * kv.kv_heads + h) * each);
        }
}

// Pieces of a workspace, each aligned to 256 bytes.
struct Carve {
    char *base;
    size_t at = 0;
    template <typename T> T *take(size_t count)
    {
        T *p = reinterpret_cast<T *>(base + at);
        at += (count * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

size_t carve(ReorderArgs &a, char *base)
{
    Carve w{base};
    a.children = w.take<int>(a.from.batch);
    a.first = w.take<int>(a.from.batch);
    a.steps = w.take<Step>(a.to.batch);
    a.counts = w.take<uint32_t>(kSegments);
    a.list = w.take<int>(a.pool.pages);
    return w.at;
}

size_t carve(CompactArgs &a, char *base)
{
    Carve w{base};
    a.low_counts = w.take<uint32_t>(kSegments);
    a.high_counts = w.take<uint32_t>(kSegments);
    a.held = w.take<int>(a.pool.pages);
    a.low = w.take<int>(a.pool.pages);
    a.high = w.take<int>(a.pool.pages);
    a.rank = w.take<int>(a.pool.pages);
    return w.at;
}

} // namespace

size_t reorder_workspace(const PoolView &pool, const TableView &from, const TableView &to)
{
    ReorderArgs a{};
    a.pool = pool, a.from = from, a.to = to;
    paged_grid(uint64_t(from.batch) + to.batch, kWave);
    return carve(a, nullptr);
}

void launch_reorder(const PoolView &pool, const TableView &from, const TableView &to,
                    const int *parents, const int *gains, uint32_t gain, int *copies,
                    char *workspace, hipStream_t stream)
{
    ReorderArgs a{};
    a.pool = pool, a.from = from, a.to = to;
    a.division = page_division(pool.page_size);
    a.parents = parents, a.gains = gains, a.gain = gain, a.copies = copies;
    a.segment = segment_of(pool.pages);
    a.segments = uint32_t((uint64_t(pool.pages) + a.segment - 1) / a.segment);
    carve(a, workspace);
    const dim3 grid = paged_grid(uint64_t(from.batch) + to.batch, kWave);
    hipLaunchKernelGGL(plan_kernel, dim3(1 + a.segments), dim3(kPlanThreads), 0, stream, a);
    check_launch("page reorder");
    hipLaunchKernelGGL(fill_kernel, grid, dim3(kWave), 0, stream, a);
    check_launch("page reorder");
}

size_t compact_workspace(const PoolView &pool, const TableView &table)
{
    CompactArgs a{};
    a.pool = pool, a.table = table;
    paged_grid(uint64_t(table.batch) + pool.pages / kWave + 1, 256);
    return carve(a, nullptr);
}

void launch_compact(const PoolView &pool, const TableView &table, uint32_t limit, int *copies,
                    uint32_t count, char *workspace, hipStream_t stream)
{
    CompactArgs a{};
    a.pool = pool, a.table = table, a.limit = limit, a.copies = copies, a.count = count;
    a.segment = segment_of(pool.pages);
    a.segments = uint32_t((uint64_t(pool.pages) + a.segment - 1) / a.segment);
    if (pool.pages <= kSpan && table.batch <= kFewHeld &&
        uint64_t(table.batch) * table.stride <= kFew && count <= kFew) {
        hipLaunchKernelGGL(compact_kernel, dim3(1), dim3(kPlanThreads), 0, stream, a);
        check_launch("page compaction");
        return;
    }
    carve(a, workspace);
    const uint64_t words = std::max(uint64_t(pool.pages), uint64_t(count) * 3);
    const uint32_t clears = uint32_t(std::min<uint64_t>((words + 255) / 256, 1024));
    hipLaunchKernelGGL(clear_kernel, dim3(clears), dim3(256), 0, stream, a);
    check_launch("page compaction");
    hipLaunchKernelGGL(count_kernel, dim3(table.batch), dim3(256), 0, stream, a);
    check_launch("page compaction");
    hipLaunchKernelGGL(sort_kernel, dim3(a.segments), dim3(kPlanThreads), 0, stream, a);
    check_launch("page compaction");
    const uint32_t most = std::min(count, pool.pages);
    hipLaunchKernelGGL(move_kernel, dim3(table.batch + (most + kWave - 1) / kWave), dim3(kWave), 0,
                       stream, a);
    check_launch("page compaction");
}

void launch_paged_copy(const PagedLayers &layers, const int *copies, uint32_t count,
                       hipStream_t stream)
{
    const PagedView &kv = layers.view;
    const uint32_t bytes = kv.head_dim * uint32_t(paged_element(kv.type));
    // a list that one launch does not cover takes several
    const uint64_t each = uint64_t(kv.kv_heads) * layers.count * 256;
    const uint32_t most = uint32_t(std::min<uint64_t>(0xffffffffull / each, count));
    require(most != 0, NUT_EINVAL, "paged cache: more rows than one launch covers");
    for (uint32_t at = 0; at < count; at += std::min(most, count - at)) {
        hipLaunchKernelGGL(copy_kernel,
                           dim3(std::min(most, count - at), kv.kv_heads, layers.count), dim3(256),
                           0, stream, layers, copies + size_t(at) * 3, bytes / 16, 2 * bytes / 16);
        check_launch("paged copy");
    }
}

} // namespace nut
