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
// a row, eight components (32 bytes of source) each. HBM bounds it: prompts of
// 8 sequences at 32 heads of 128, fp16, 421 MB in 83 us (5.1 TB/s; a 4 GiB copy
// moves 4.75). One token each of 64 sequences is a launch, 4.8 us.
template <int TYPE>
__global__ __launch_bounds__(256) void append_kernel(
    PagedView kv, PagedSeqs s, const float *__restrict__ keys, const float *__restrict__ values,
    size_t rows, size_t row_stride, size_t head_stride, const int *__restrict__ starts,
    uint32_t each, uint32_t max_new, PagedHistory history, const int *__restrict__ firsts,
    int *new_lengths, uint32_t touched)
{
    const uint32_t id = blockIdx.x;
    const uint32_t c = id % touched, h = id / touched % kv.kv_heads;
    const uint32_t b = id / touched / kv.kv_heads;
    const bool leader = threadIdx.x == 0 && h == 0 && c == 0;

    const int length = s.lengths[b];
    const int64_t from = starts == nullptr ? int64_t(b) * each : starts[b];
    int64_t gain = starts == nullptr ? int64_t(each) : starts[b + 1] - from;
    const int bad = append_error(length, from, gain, max_new, rows, s.max_length);
    if (bad != 0)
        gain = 0;
    if (leader) {
        if (bad != 0)
            paged_flag(kv.status, bad);
        if (new_lengths != nullptr)
            new_lengths[b] = length + int(gain);
    }
    if (gain == 0)
        return;

    const uint32_t n = uint32_t(length), ps = kv.page_size;
    const AppendSpan span = append_span(n, uint32_t(gain), c, ps, kv.division);
    const uint32_t index = span.index, begin = span.begin, end = span.end;
    if (begin == end)
        return;
    constexpr uint32_t kSize = TYPE == NUT_F32 ? 4 : 2;
    const uint32_t tpr = kv.head_dim / 8, part = threadIdx.x % tpr, group = threadIdx.x / tpr;
    const uint32_t groups = blockDim.x / tpr;
    // the first row of a group beside the table, and the page's bounds beside the
    // rows' stores
    float k[8] = {}, v[8] = {};
    const auto fetch = [&](uint32_t r) {
        const size_t source = (size_t(from) + (r - n)) * row_stride + h * head_stride + part * 8;
        load8<NUT_F32>(reinterpret_cast<const char *>(keys + source), k);
        load8<NUT_F32>(reinterpret_cast<const char *>(values + source), v);
    };
    const bool first = group < groups && begin + group < end;
    if (first)
        fetch(begin + group);
    const size_t page = paged_row(kv, s, b, index, 0, h);
    if (history.weights != nullptr) {
        const size_t at = (size_t(b) * kv.kv_heads + h) * history.stride;
        const int position = firsts == nullptr ? length : firsts[b];
        for (uint32_t r = begin + threadIdx.x; r < end; r += blockDim.x) {
            history.weights[at + r] = 0.0f;
            history.positions[at + r] = position + int(r - n);
        }
    }
    if (page == kNoRow)
        return;
    char *bounds = kv.bounds + (size_t(s.table[size_t(b) * s.table_stride + index]) * kv.kv_heads +
                                h) * 2 * kv.head_dim * kSize + threadIdx.x * 8 * kSize;
    float least[8], most[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        least[i] = INFINITY, most[i] = -INFINITY;
    if (kv.bounds != nullptr && threadIdx.x < tpr && index * ps < n) {
        load8<TYPE>(bounds, least);
        load8<TYPE>(bounds + kv.head_dim * kSize, most);
    }
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        lo[i] = INFINITY, hi[i] = -INFINITY;
    if (first)
        for (uint32_t r = begin + group; r < end; r += groups) {
            if (r != begin + group)
                fetch(r);
            const size_t to = page + size_t(r - index * ps) * kv.slot_stride + part * 8 * kSize;
            store8<TYPE>(kv.keys + to, k);
            store8<TYPE>(kv.values + to, v);
#pragma unroll
            for (int i = 0; i < 8; i++)
                lo[i] = lower(lo[i], k[i]), hi[i] = upper(hi[i], k[i]);
        }
    if (kv.bounds == nullptr)
        return;
    // The upper half of the groups hands its bounds to the lower one, and so on:
    // 71 tokens each of 3 sequences, 4 heads of 64, 6.7 us where one group that
    // read all the others' took 12.1.
    __shared__ float low[256][8], high[256][8];
    const uint32_t used = min(groups, end - begin);
    for (uint32_t half = used == 1 ? 0 : 1u << (31 - __clz(used - 1)); half > 0; half /= 2) {
        if (group >= half && group < min(2 * half, used))
#pragma unroll
            for (int i = 0; i < 8; i++)
                low[threadIdx.x][i] = lo[i], high[threadIdx.x][i] = hi[i];
        __syncthreads();
        if (group < half && group + half < used)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                lo[i] = lower(lo[i], low[threadIdx.x + half * tpr][i]);
                hi[i] = upper(hi[i], high[threadIdx.x + half * tpr][i]);
            }
    }
    if (threadIdx.x >= tpr) // a workgroup has tpr threads at least
        return;
#pragma unroll
    for (int i = 0; i < 8; i++)
        least[i] = lower(least[i], lo[i]), most[i] = upper(most[i], hi[i]);
    store8<TYPE>(bounds, least);
    store8<TYPE>(bounds + kv.head_dim * kSize, most);
}

// ------------------------------------------------------ the k-th largest --

constexpr int kBits = 8, kBins = 1 << kBits;

struct RankScratch {
    alignas(16) uint32_t bins[kBins];
    uint32_t any[2], lacked[2]; // bits that some key has, and that some key lacks
    uint32_t bin, above, count;
    uint32_t places[130]; // of each wave's run of 64 keys, and their sum
};

template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ uint32_t dpp_bits(uint32_t v, uint32_t fill)
{
    return uint32_t(__builtin_amdgcn_update_dpp(int(fill), int(v), CTRL, ROWS, 0xF, false));
}

// Bits that any lane of the wave has, in lane 63.
__device__ __forceinline__ uint32_t any_bits(uint32_t v)
{
    v |= dpp_bits<kDppQuadSwap1>(v, 0);
    v |= dpp_bits<kDppQuadSwap2>(v, 0);
    v |= dpp_bits<kDppRowHalfMirror>(v, 0);
    v |= dpp_bits<kDppRowMirror>(v, 0);
    v |= dpp_bits<kDppRowBcast15, 0xA>(v, 0);
    return v | dpp_bits<kDppRowBcast31, 0xC>(v, 0);
}

// The largest of a wave's values, none below -1, in lane 63.
__device__ __forceinline__ int largest(int v)
{
    v = max(v, int(dpp_bits<kDppQuadSwap1>(v, ~0u)));
    v = max(v, int(dpp_bits<kDppQuadSwap2>(v, ~0u)));
    v = max(v, int(dpp_bits<kDppRowHalfMirror>(v, ~0u)));
    v = max(v, int(dpp_bits<kDppRowMirror>(v, ~0u)));
    v = max(v, int(dpp_bits<kDppRowBcast15, 0xA>(v, ~0u)));
    return max(v, int(dpp_bits<kDppRowBcast31, 0xC>(v, ~0u)));
}

// Sum of this lane's value and those of the lanes below it.
__device__ __forceinline__ uint32_t running_sum(uint32_t v)
{
    constexpr int kRowShift = 0x110; // lane i of a row of 16 from lane i - n
    v += dpp_bits<kRowShift + 1>(v, 0);
    v += dpp_bits<kRowShift + 2>(v, 0);
    v += dpp_bits<kRowShift + 4>(v, 0);
    v += dpp_bits<kRowShift + 8>(v, 0);
    v += dpp_bits<kDppRowBcast15, 0xA>(v, 0);
    return v + dpp_bits<kDppRowBcast31, 0xC>(v, 0);
}

// Lanes below this one in a ballot.
__device__ __forceinline__ uint32_t rank_in(uint64_t mask)
{
    return __builtin_amdgcn_mbcnt_hi(uint32_t(mask >> 32),
                                     __builtin_amdgcn_mbcnt_lo(uint32_t(mask), 0));
}

// Keys 0 to n - 1 of a workgroup, EACH a thread in registers (key
// e THREADS + thread), and segment after segment of so many, read anew each
// time by `load`, where there are more.
template <typename K, int THREADS, int EACH, typename Load> struct Keys {
    static constexpr uint32_t kSegment = THREADS * EACH;
    const Load &load;
    uint32_t n;
    K key[EACH];

    __device__ __forceinline__ uint32_t index(uint32_t segment, int e) const
    {
        return segment + e * THREADS + threadIdx.x;
    }
    __device__ __forceinline__ void open(uint32_t segment)
    {
        if (n > kSegment)
#pragma unroll
            for (int e = 0; e < EACH; e++)
                key[e] = index(segment, e) < n ? load(index(segment, e)) : K(0);
    }
    template <typename Use> __device__ __forceinline__ void each(Use use)
    {
        for (uint32_t segment = 0; segment < n; segment += kSegment) {
            open(segment);
#pragma unroll
            for (int e = 0; e < EACH; e++)
                if (index(segment, e) < n)
                    use(key[e]);
        }
    }
};

// Finds the threshold T and the number of ties such that the k largest keys
// (1 <= k < n), ties to the lowest index, are the keys over T and the first
// `ties` keys equal to T. A radix search from the first bit in which the keys
// differ, 8 bits a pass, which ends at the first digit whose keys are all
// taken: two or three passes of scores that differ in their leading bits.
// Every thread of the workgroup calls it, with sc.bins, any and lacked zero
// and a barrier behind that; it ends at a barrier.
template <typename K, int THREADS, int EACH, typename Load>
__device__ __forceinline__ void kth_largest(Keys<K, THREADS, EACH, Load> &keys, uint32_t k,
                                            RankScratch &sc, K &threshold, uint32_t &ties)
{
    constexpr int kWidth = 8 * sizeof(K);
    const uint32_t lane = threadIdx.x & (kWave - 1);
    K any = 0, all = K(~K(0));
    keys.each([&](K key) { any |= key, all &= key; });
#pragma unroll
    for (int w = 0; w < kWidth / 32; w++) {
        const uint32_t has = any_bits(uint32_t(any >> (32 * w)));
        const uint32_t lacks = any_bits(uint32_t(~all >> (32 * w)));
        if (lane == kWave - 1) {
            atomicOr(&sc.any[w], has);
            atomicOr(&sc.lacked[w], lacks);
        }
    }
    __syncthreads();
    any = 0;
    K differ = 0;
#pragma unroll
    for (int w = 0; w < kWidth / 32; w++) {
        any |= K(sc.any[w]) << (32 * w);
        differ |= K(sc.any[w] & sc.lacked[w]) << (32 * w);
    }
    if (differ == 0) {
        threshold = any;
        ties = k;
        return;
    }
    int open = 64 - __clzll((unsigned long long)differ); // bits not yet decided
    K prefix = open >= kWidth ? K(0) : K(any >> open << open);
    uint32_t left = k;
    while (true) {
        const int shift = max(0, open - kBits);
        const uint32_t mask = (1u << (open - shift)) - 1;
        keys.each([&](K key) {
            if (open >= kWidth || (K(key ^ prefix) >> open) == 0)
                atomicAdd(&sc.bins[uint32_t(key >> shift) & mask], 1u);
        });
        __syncthreads();
        if (threadIdx.x < kWave) {
            // lane l holds bins 255 - 4 l down to 252 - 4 l: from the highest
            uint4 *at = reinterpret_cast<uint4 *>(sc.bins) + (kWave - 1 - lane);
            const uint4 bins = *at;
            *at = make_uint4(0, 0, 0, 0); // for the next pass
            const uint32_t own = bins.x + bins.y + bins.z + bins.w;
            const uint32_t scan = running_sum(own);
            if (scan >= left && scan - own < left) {
                const uint32_t size[4] = {bins.w, bins.z, bins.y, bins.x};
                uint32_t above = scan - own, bin = 255 - 4 * lane, count = size[0];
#pragma unroll
                for (int i = 1; i < 4; i++)
                    if (above + count < left)
                        above += count, bin--, count = size[i];
                sc.bin = bin, sc.above = above, sc.count = count;
            }
        }
        __syncthreads();
        prefix |= K(sc.bin) << shift;
        left -= sc.above;
        if (sc.count == left || shift == 0) {
            threshold = prefix;
            ties = sc.count == left ? 0xffffffffu : left;
            return;
        }
        open = shift;
        // sc.bin and its neighbours are written again behind the next barrier
    }
}

// place[e] becomes the number of set flags before flag e of this thread, in the
// order of keys, `base` growing by all of them. Flags are counts of two kinds
// in halves of a word. Every thread calls it; sc.places may be in use until
// the first barrier only.
template <int THREADS, int EACH>
__device__ __forceinline__ void places_of(const uint32_t (&flag)[EACH], uint32_t (&place)[EACH],
                                          uint32_t &base, RankScratch &sc)
{
    constexpr uint32_t kWaves = THREADS / kWave, kRuns = kWaves * EACH;
    static_assert(kRuns <= 128, "two runs a lane");
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    uint32_t sum = 0; // of lane e's run
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const uint64_t low = __ballot(flag[e] & 0xffffu), high = __ballot(flag[e] >> 16);
        place[e] = rank_in(low) | rank_in(high) << 16;
        if (lane == uint32_t(e))
            sum = __popcll(low) | uint32_t(__popcll(high)) << 16;
    }
    __syncthreads();
    if (lane < EACH)
        sc.places[lane * kWaves + wave] = sum;
    __syncthreads();
    if (threadIdx.x < kWave) {
        const uint32_t a = 2 * lane < kRuns ? sc.places[2 * lane] : 0;
        const uint32_t z = 2 * lane + 1 < kRuns ? sc.places[2 * lane + 1] : 0;
        const uint32_t scan = running_sum(a + z);
        sc.places[2 * lane] = scan - a - z;
        sc.places[2 * lane + 1] = scan - z;
        if (lane == kWave - 1)
            sc.places[128] = scan;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; e++)
        place[e] += base + sc.places[e * kWaves + wave];
    base += sc.places[128];
}

// ---------------------------------------------------------------- select --

// A partner's value among the lanes of a page: for O = 2 and 1 the lane O away,
// for 8 and 4 the mirror image in 2 O lanes, which lies O away in the bit that
// counts and has not been told apart in the others yet.
template <int O> __device__ __forceinline__ uint32_t partner(uint32_t v)
{
    if constexpr (O == 16)
        return __shfl_xor(v, 16);
    else
        return dpp_bits<(O == 8   ? kDppRowMirror
                         : O == 4 ? kDppRowHalfMirror
                         : O == 2 ? kDppQuadSwap2
                                  : kDppQuadSwap1)>(v, 0);
}

template <int O> __device__ __forceinline__ uint64_t partner_bits(uint64_t v)
{
    return uint64_t(partner<O>(uint32_t(v >> 32))) << 32 | partner<O>(uint32_t(v));
}

// Sums over the 2 O lanes of a page: while a lane holds several heads it trades
// half of them for the other half's part, then it adds. `head` becomes the
// first head that is left, of HELD / (2 O) or one.
template <int O, int HELD>
__device__ __forceinline__ void sum_lanes(double *sum, uint32_t part, uint32_t &head)
{
    if constexpr (O > 0) {
        if constexpr (HELD > 1) {
            const bool up = part & O;
#pragma unroll
            for (int j = 0; j < HELD / 2; j++) {
                const double give = up ? sum[j] : sum[j + HELD / 2];
                const double keep = up ? sum[j + HELD / 2] : sum[j];
                sum[j] = keep + __builtin_bit_cast(
                                    double, partner_bits<O>(__builtin_bit_cast(uint64_t, give)));
            }
            head += up ? HELD / 2 : 0;
            sum_lanes<O / 2, HELD / 2>(sum, part, head);
        } else {
            sum[0] += __builtin_bit_cast(
                double, partner_bits<O>(__builtin_bit_cast(uint64_t, sum[0])));
            sum_lanes<O / 2, 1>(sum, part, head);
        }
    }
}

template <int O> __device__ __forceinline__ uint64_t best_of_lanes(uint64_t v)
{
    if constexpr (O > 0) {
        const uint64_t other = partner_bits<O>(v);
        return best_of_lanes<O / 2>(other > v ? other : v);
    }
    return v;
}

// Order-preserving image of a score; a NaN ranks above every number, the
// pages that are always read above both.
__device__ __forceinline__ uint64_t score_key(double v)
{
    if (v != v)
        return ~0ull - 1;
    const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0); // -0 ranks as 0
    return u >> 63 ? ~u : u | (1ull << 63);
}

// A component's part of a page's score, max(q lo, q hi), of finite or infinite
// bounds; not a number where a product is not (one of them, of a query of 0 and
// an infinite bound).
__device__ __forceinline__ double score_part(float q, float lo, float hi)
{
    const double a = double(q) * double(lo), b = double(q) * double(hi);
    return a > b || a != a ? a : b;
}

// Eight components' part.
template <int TYPE>
__device__ __forceinline__ double score_of(const float *query, const char *bounds,
                                           uint32_t head_dim)
{
    constexpr uint32_t kSize = TYPE == NUT_F32 ? 4 : 2;
    float q[8], lo[8], hi[8];
    load8<NUT_F32>(reinterpret_cast<const char *>(query), q);
    load8<TYPE>(bounds, lo);
    load8<TYPE>(bounds + head_dim * kSize, hi);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 8; i++)
        sum += score_part(q[i], lo[i], hi[i]);
    return sum;
}

// Scores of every page, up to four heads to a KV head: LANES lanes, head_dim / 8
// of them with work, hold eight components of a page's bounds each. For a page
//   sum_d max(q_d lo_d, q_d hi_d) = sum_d max(q_d, 0) hi_d + min(q_d, 0) lo_d,
// two multiply-adds a component in 64 bits, of which one adds zero: the answer
// is whole numbers, and in 32 bits, or with terms that only cancel, rounding
// would choose among near or equal pages. An infinite bound that the query does
// not meet makes the term that adds zero no number: such sums are made anew from
// the definition, the same additions without those terms. What bounds it is
// instructions: 16 fp64 ones a head and eight to bring them together, for 64
// bytes a lane.
template <int TYPE, int GH, uint32_t LANES>
__global__ __launch_bounds__(256) void page_scores_kernel(PagedView kv, PagedSeqs s,
                                                          const float *__restrict__ query,
                                                          size_t query_stride, uint32_t heads,
                                                          uint32_t blocks, uint32_t width,
                                                          uint64_t *__restrict__ scores)
{
    constexpr uint32_t kSize = TYPE == NUT_F32 ? 4 : 2;
    const uint32_t id = blockIdx.x, c = id % blocks, h = id / blocks % kv.kv_heads;
    const uint32_t b = id / blocks / kv.kv_heads;
    const uint32_t index = c * (256 / LANES) + threadIdx.x / LANES, part = threadIdx.x % LANES;
    const uint32_t group = heads / kv.kv_heads;
    const bool works = part * 8 < kv.head_dim;
    const float *own = query + b * query_stride + size_t(h) * group * kv.head_dim + part * 8;
    // the query and the table beside the length: what lies behind it is not used
    double up[GH][8], down[GH][8]; // max(q, 0) and min(q, 0)
#pragma unroll
    for (int j = 0; j < GH; j++) {
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (works && uint32_t(j) < group)
            load8<NUT_F32>(reinterpret_cast<const char *>(own + size_t(j) * kv.head_dim), v);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // a query component that is not a number stays one
            up[j][i] = double(v[i] <= 0.0f ? 0.0f : v[i]);
            down[j][i] = double(v[i] >= 0.0f ? 0.0f : v[i]);
        }
    }
    const int page = index < width ? s.table[size_t(b) * s.table_stride + index] : -1;
    const uint32_t n = paged_length(kv, s, b, threadIdx.x == 0 && h == 0 && c == 0);
    const uint32_t count = n == 0 ? 0 : page_of(kv, n - 1) + 1;
    if (index >= count)
        return;
    const bool good = page_in(page, kv.pages);
    if (!good && part == 0)
        paged_flag(kv.status, kBadPage);
    float lo[8] = {0, 0, 0, 0, 0, 0, 0, 0}, hi[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    const char *at = kv.bounds + (size_t(good ? page : 0) * kv.kv_heads + h) * 2 * kv.head_dim *
                                     kSize + part * 8 * kSize;
    if (good && works) {
        load8<TYPE>(at, lo);
        load8<TYPE>(at + kv.head_dim * kSize, hi);
    }
    double sum[GH];
#pragma unroll
    for (int j = 0; j < GH; j++)
        sum[j] = 0.0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const double high = hi[i], low = lo[i];
#pragma unroll
        for (int j = 0; j < GH; j++)
            sum[j] = fma(down[j][i], low, fma(up[j][i], high, sum[j]));
    }
    bool odd = false;
#pragma unroll
    for (int j = 0; j < GH; j++)
        odd = odd || sum[j] != sum[j];
    if (odd) // the query and the bounds once more: held till here, they cost waves
#pragma unroll
        for (int j = 0; j < GH; j++) {
            const double x = works && uint32_t(j) < group
                                 ? score_of<TYPE>(own + size_t(j) * kv.head_dim, at, kv.head_dim)
                                 : 0.0;
            sum[j] = sum[j] != sum[j] ? x : sum[j];
        }
    uint32_t head = 0;
    sum_lanes<LANES / 2, GH>(sum, part, head);
    constexpr int kLeft = GH > int(LANES) ? GH / int(LANES) : 1;
    uint64_t best = 0;
#pragma unroll
    for (int j = 0; j < kLeft; j++) {
        const uint64_t key = score_key(sum[j]);
        if (head + j < group && key > best)
            best = key;
    }
    best = best_of_lanes<LANES / 2>(best);
    if (part == 0) // a bad page below all others
        scores[(size_t(b) * kv.kv_heads + h) * width + index] = good ? best : 0;
}

// What a page's infinite bounds add to its score: infinities, and no number
// where they meet a query of 0.
template <int TYPE>
__device__ __forceinline__ double unbounded_part(const float *query, const char *bounds,
                                                 uint32_t head_dim)
{
    constexpr uint32_t kSize = TYPE == NUT_F32 ? 4 : 2;
    double sum = 0.0;
#pragma unroll 1
    for (uint32_t d = 0; d < head_dim; d += 8) {
        float q[8], lo[8], hi[8];
        load8<NUT_F32>(reinterpret_cast<const char *>(query + d), q);
        load8<TYPE>(bounds + d * kSize, lo);
        load8<TYPE>(bounds + (head_dim + d) * kSize, hi);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const double part = score_part(q[i], lo[i], hi[i]);
            if (fmaxf(fabsf(lo[i]), fabsf(hi[i])) == INFINITY && !(fabs(part) < INFINITY))
                sum += part;
        }
    }
    return sum;
}

typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// The sums of page_scores_mfma_kernel anew, product by product, with infinite
// bounds left out; whether the lane's components of its page have one. `own` is
// the query of the lane's head.
template <int TYPE>
__device__ __forceinline__ bool bounded_sums(const float *own, bool valid, const char *bounds,
                                             bool good, uint32_t head_dim, f64x4 &above,
                                             f64x4 &below)
{
    constexpr uint32_t kSize = TYPE == NUT_F32 ? 4 : 2;
    const uint32_t j = (threadIdx.x & (kWave - 1)) / 16;
    bool unbounded = false;
    above = below = f64x4{0, 0, 0, 0};
#pragma unroll 1
    for (uint32_t step = 0; step < (head_dim + 63) / 64 * 2; step++) {
        const uint32_t d = step / 2 * 64 + 16 * j + step % 2 * 8;
        float q[8] = {0, 0, 0, 0, 0, 0, 0, 0}, lo[8] = {0, 0, 0, 0, 0, 0, 0, 0},
              hi[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (valid && d < head_dim)
            load8<NUT_F32>(reinterpret_cast<const char *>(own + d), q);
        if (good && d < head_dim) {
            load8<TYPE>(bounds + d * kSize, lo);
            load8<TYPE>(bounds + (head_dim + d) * kSize, hi);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const bool low = fabsf(lo[i]) == INFINITY, high = fabsf(hi[i]) == INFINITY;
            unbounded = unbounded || low || high;
            above = __builtin_amdgcn_mfma_f64_16x16x4f64(
                double(high ? 0.0f : hi[i]), double(q[i] <= 0.0f ? 0.0f : q[i]), above, 0, 0, 0);
            below = __builtin_amdgcn_mfma_f64_16x16x4f64(
                double(low ? 0.0f : lo[i]), double(q[i] >= 0.0f ? 0.0f : q[i]), below, 0, 0, 0);
        }
    }
    return unbounded;
}

// The same for more than four heads to a KV head, on v_mfma_f64_16x16x4f64: a
// wave takes 16 pages (rows) and 16 heads (columns), and sums over 64
// components at a time, max(q, 0) hi and min(q, 0) lo apart. Lane 16 j + c
// loads components 16 j to 16 j + 15 of page c, whose n-th is the j-th of
// four in step n; the query comes from shared memory, [sign][component][head].
// Scores of pages 4 i + j and head c come out as element i of that lane. 49,140
// pages of 64 components and 8 heads take 10.9 us, which neither their 12.6 MB
// (2.0 us) nor their matrix instructions (32 of 64 cycles a tile, 3 tiles a
// SIMD: 2.7 us of pipe by its counter) bound: all waves are there at once, four
// to a SIMD, and wait for the length, the bounds and the staged query before
// any of them multiplies. No bank of shared memory is asked for twice (counter
// 0). A tile with a sum that is no number is summed anew without infinite
// bounds, which a query of the other sign would make one, and what they add is
// found from the definition.
template <int TYPE>
__global__ __launch_bounds__(256) void page_scores_mfma_kernel(PagedView kv, PagedSeqs s,
                                                               const float *__restrict__ query,
                                                               size_t query_stride,
                                                               uint32_t heads, uint32_t blocks,
                                                               uint32_t width,
                                                               uint64_t *__restrict__ scores)
{
    constexpr uint32_t kSize = TYPE == NUT_F32 ? 4 : 2;
    __shared__ double qs[2][64][16];
    const uint32_t id = blockIdx.x, block = id % blocks, h = id / blocks % kv.kv_heads;
    const uint32_t b = id / blocks / kv.kv_heads;
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const uint32_t j = lane / 16, c = lane % 16, group = heads / kv.kv_heads;
    const uint32_t base = block * 64 + wave * 16;
    // the table beside the length: what lies behind it is not used
    int page = base + c < width ? s.table[size_t(b) * s.table_stride + base + c] : -1;
    const float *rows = query + b * query_stride + size_t(h) * group * kv.head_dim;
    const uint32_t head = threadIdx.x % 16, d = threadIdx.x / 16 * 4;
    const auto fetch = [&](uint32_t g, uint32_t slab) {
        return g + head < group && slab + d < kv.head_dim
                   ? *reinterpret_cast<const f32x4 *>(rows + size_t(g + head) * kv.head_dim +
                                                      slab + d)
                   : f32x4{0, 0, 0, 0};
    };
    f32x4 x = fetch(0, 0);
    const uint32_t n = paged_length(kv, s, b, threadIdx.x == 0 && h == 0 && block == 0);
    asm volatile("" : "+v"(page), "+v"(x));
    const uint32_t count = n == 0 ? 0 : page_of(kv, n - 1) + 1;
    if (block * 64 >= count)
        return;
    const bool good = page_in(page, kv.pages) && base + c < count;
    if (!good && base + c < count)
        paged_flag(kv.status, kBadPage);
    const uint32_t there = uint32_t(__ballot(good)); // bit c: page c
    const char *bounds = kv.bounds + (size_t(good ? page : 0) * kv.kv_heads + h) * 2 *
                                         kv.head_dim * kSize;
    uint64_t best[4] = {0, 0, 0, 0};
    for (uint32_t g = 0; g < group; g += 16) {
        f64x4 above{0, 0, 0, 0}, below{0, 0, 0, 0}; // by hi, by lo
        for (uint32_t slab = 0; slab < kv.head_dim; slab += 64) {
            if (g + slab != 0)
                x = fetch(g, slab);
            float hi[16], lo[16];
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
                float low[8] = {0, 0, 0, 0, 0, 0, 0, 0}, high[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (good && slab + 16 * j + e < kv.head_dim) {
                    load8<TYPE>(bounds + (slab + 16 * j + e) * kSize, low);
                    load8<TYPE>(bounds + (kv.head_dim + slab + 16 * j + e) * kSize, high);
                }
#pragma unroll
                for (int i = 0; i < 8; i++)
                    lo[e + i] = low[i], hi[e + i] = high[i];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; i++) {
                // a query component that is not a number stays one
                qs[0][d + i][head] = double(x[i] <= 0.0f ? 0.0f : x[i]);
                qs[1][d + i][head] = double(x[i] >= 0.0f ? 0.0f : x[i]);
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 16; e++) {
                above = __builtin_amdgcn_mfma_f64_16x16x4f64(double(hi[e]), qs[0][16 * j + e][c],
                                                             above, 0, 0, 0);
                below = __builtin_amdgcn_mfma_f64_16x16x4f64(double(lo[e]), qs[1][16 * j + e][c],
                                                             below, 0, 0, 0);
            }
        }
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 4; i++)
            odd = odd || above[i] + below[i] != above[i] + below[i];
        if (__any(odd)) {
            const float *own = rows + size_t(g + c < group ? g + c : 0) * kv.head_dim;
            const uint64_t lanes = __ballot(
                bounded_sums<TYPE>(own, g + c < group, bounds, good, kv.head_dim, above, below));
            const uint32_t which = uint32_t(lanes | lanes >> 16 | lanes >> 32 | lanes >> 48);
#pragma unroll 1
            for (uint32_t p = j; p < 16; p += 4) {
                const int its = __shfl(page, int(p));
                double more = 0.0;
                if (which >> p & 1 && g + c < group)
                    more = unbounded_part<TYPE>(
                        own, kv.bounds + (size_t(its) * kv.kv_heads + h) * 2 * kv.head_dim * kSize,
                        kv.head_dim);
#pragma unroll
                for (uint32_t i = 0; i < 4; i++)
                    above[i] += i == p / 4 ? more : 0.0;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint64_t key = g + c < group ? score_key(above[i] + below[i]) : 0;
            best[i] = key > best[i] ? key : best[i];
        }
    }
    uint64_t *out = scores + (size_t(b) * kv.kv_heads + h) * width;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint64_t key = best_of_lanes<8>(best[i]);
        const uint32_t p = 4 * i + j;
        if (c == 0 && base + p < count) // a bad page below all others
            out[base + p] = there >> p & 1 ? key : 0;
    }
}

// A workgroup per (sequence, KV head): the `top` best of its pages. Barriers and
// the first read bound it: 6.3 us for 1,024 pages each of 64 KV heads.
__global__ __launch_bounds__(256) void choose_pages_kernel(PagedView kv, PagedSeqs s,
                                                           const uint64_t *__restrict__ scores,
                                                           uint32_t width, uint32_t top,
                                                           uint32_t first, uint32_t last,
                                                           int *__restrict__ selected)
{
    constexpr int kEach = 8;
    __shared__ RankScratch sc;
    const uint32_t id = blockIdx.x, h = id % kv.kv_heads, b = id / kv.kv_heads;
    const uint64_t *mine = scores + (size_t(b) * kv.kv_heads + h) * width;
    // the first scores beside the length: those behind it are not used
    uint64_t early[kEach];
#pragma unroll
    for (int e = 0; e < kEach; e++)
        early[e] = e * 256 + threadIdx.x < width ? mine[e * 256 + threadIdx.x] : 0;
    sc.bins[threadIdx.x] = 0;
    if (threadIdx.x < 2)
        sc.any[threadIdx.x] = sc.lacked[threadIdx.x] = 0;
    const uint32_t n = paged_length(kv, s, b, threadIdx.x == 0 && h == 0);
    const uint32_t count = n == 0 ? 0 : page_of(kv, n - 1) + 1;
    int *out = selected + (size_t(b) * kv.kv_heads + h) * top;
    if (count <= top) {
        for (uint32_t i = threadIdx.x; i < top; i += 256)
            out[i] = i < count ? int(i) : -1;
        return;
    }
    const auto key_of = [&](uint32_t i, uint64_t score) -> uint64_t {
        return i < first || i >= count - last ? ~0ull : score;
    };
    const auto load = [&](uint32_t i) { return key_of(i, mine[i]); };
    Keys<uint64_t, 256, kEach, decltype(load)> keys{load, count, {}};
#pragma unroll
    for (int e = 0; e < kEach; e++)
        keys.key[e] = key_of(e * 256 + threadIdx.x, early[e]);
    __syncthreads();
    uint64_t threshold;
    uint32_t ties;
    kth_largest(keys, top, sc, threshold, ties);

    uint32_t at = 0, met = 0;
    for (uint32_t segment = 0; segment < count; segment += keys.kSegment) {
        keys.open(segment);
        uint32_t flag[kEach], place[kEach];
        bool kept[kEach];
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            const bool in = keys.index(segment, e) < count;
            kept[e] = in && keys.key[e] >= threshold;
            flag[e] = in && keys.key[e] == threshold;
        }
        if (ties != 0xffffffffu) {
            places_of<256, kEach>(flag, place, met, sc);
#pragma unroll
            for (int e = 0; e < kEach; e++)
                kept[e] = kept[e] && (flag[e] == 0 || place[e] < ties);
        }
#pragma unroll
        for (int e = 0; e < kEach; e++)
            flag[e] = kept[e];
        places_of<256, kEach>(flag, place, at, sc);
#pragma unroll
        for (int e = 0; e < kEach; e++)
            if (kept[e])
                out[place[e]] = int(keys.index(segment, e));
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

// A workgroup per (sequence, KV head) decides what stays: to[r] is the r-th
// row below the budget that goes, from[r] the r-th beyond it that stays (`list`
// at most), and counts how many there are. Weights and positions of up to eight rows a
// thread are read once; then barriers bound it: 9 us for 1,040 rows each of 64
// KV heads, 12 us for 8,192 each of 128.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void plan_eviction_kernel(PagedView kv, PagedSeqs s,
                                                                PagedHistory history,
                                                                uint32_t budget, uint32_t first,
                                                                uint32_t last, uint32_t list,
                                                                int *new_lengths,
                                                                int *__restrict__ to,
                                                                int *__restrict__ from,
                                                                int *__restrict__ counts)
{
    constexpr int kEach = 8;
    __shared__ RankScratch sc;
    __shared__ int newest_of[THREADS / kWave];
    const uint32_t id = blockIdx.x, h = id % kv.kv_heads, b = id / kv.kv_heads;
    const bool leader = threadIdx.x == 0 && h == 0;
    const size_t at = (size_t(b) * kv.kv_heads + h) * history.stride;
    const float *weights = history.weights + at;
    const int *positions = history.positions + at;
    // the first rows beside the length, which max_length bounds
    float w[kEach];
    int p[kEach];
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        const uint32_t i = e * THREADS + threadIdx.x;
        w[e] = i < s.max_length ? weights[i] : 0.0f;
        p[e] = i < s.max_length ? positions[i] : 0;
    }
    if (threadIdx.x < kBins)
        sc.bins[threadIdx.x] = 0;
    if (threadIdx.x < 2)
        sc.any[threadIdx.x] = sc.lacked[threadIdx.x] = 0;
    const uint32_t n = paged_length(kv, s, b, leader);
    if (leader)
        new_lengths[b] = n > budget ? int(budget) : s.lengths[b];
    if (n <= budget) {
        if (threadIdx.x == 0)
            counts[id] = 0;
        return;
    }
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    int newest = -1;
#pragma unroll
    for (int e = 0; e < kEach; e++)
        if (e * THREADS + threadIdx.x < n)
            newest = max(newest, p[e]);
    for (uint32_t i = kEach * THREADS + threadIdx.x; i < n; i += THREADS)
        newest = max(newest, positions[i]);
    newest = largest(newest);
    if (lane == kWave - 1)
        newest_of[wave] = newest;
    __syncthreads();
    newest = newest_of[0];
#pragma unroll
    for (int v = 1; v < THREADS / kWave; v++)
        newest = max(newest, newest_of[v]);
    const int64_t recent = int64_t(newest) - int64_t(last);
    const auto key_of = [&](int position, float weight) -> uint32_t {
        return position < int64_t(first) || position > recent ? 0xffffffffu : weight_key(weight);
    };
    const auto load = [&](uint32_t i) { return key_of(positions[i], weights[i]); };
    Keys<uint32_t, THREADS, kEach, decltype(load)> keys{load, n, {}};
#pragma unroll
    for (int e = 0; e < kEach; e++)
        keys.key[e] = key_of(p[e], w[e]);
    uint32_t threshold, ties;
    kth_largest(keys, budget, sc, threshold, ties);

    // holes in the lower halves of words, rows to move in the upper ones: each
    // segment has at most 2^13 of them
    uint32_t met = 0, holes = 0, moved = 0;
    int *hole_at = to + size_t(id) * list, *source = from + size_t(id) * list;
    for (uint32_t segment = 0; segment < n; segment += keys.kSegment) {
        keys.open(segment);
        uint32_t flag[kEach], place[kEach];
        bool kept[kEach];
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            const bool in = keys.index(segment, e) < n;
            kept[e] = in && keys.key[e] >= threshold;
            flag[e] = in && keys.key[e] == threshold;
        }
        if (ties != 0xffffffffu) {
            places_of<THREADS, kEach>(flag, place, met, sc);
#pragma unroll
            for (int e = 0; e < kEach; e++)
                kept[e] = kept[e] && (flag[e] == 0 || place[e] < ties);
        }
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            const uint32_t i = keys.index(segment, e);
            flag[e] = i >= n ? 0 : i < budget ? !kept[e] : uint32_t(kept[e]) << 16;
        }
        uint32_t both = 0;
        places_of<THREADS, kEach>(flag, place, both, sc);
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            if (flag[e] == 1)
                hole_at[holes + (place[e] & 0xffffu)] = int(keys.index(segment, e));
            else if (flag[e] != 0)
                source[moved + (place[e] >> 16)] = int(keys.index(segment, e));
        }
        holes += both & 0xffffu;
        moved += both >> 16;
    }
    if (threadIdx.x == 0)
        counts[id] = int(moved);
}

// A workgroup per (sequence, KV head, 256 entries of its list): a thread an
// entry finds where the row lies and takes its weight and position along, then
// head_dim / 8 threads a row copy rows. Sources lie beyond the budget and are
// only read, so the order of workgroups does not matter; the bounds of a page
// whose entries begin in one workgroup's part and end in another's are the
// first one's. HBM bounds it: 205 MB of rows from anywhere to anywhere in 46 us
// (4.5 TB/s) where 128 KV heads of up to 8,192 rows keep 2,048. With bounds it
// does not: the threads of a page read its entries, the table and the keys once
// more, one row after another, and the whole call takes 315 us for 64.5 (16.8
// for 14.0 where 64 heads are up to 16 rows over 1,024).
template <int TYPE>
__global__ __launch_bounds__(256) void move_rows_kernel(PagedView kv, PagedSeqs s,
                                                        PagedHistory history, uint32_t list,
                                                        uint32_t blocks,
                                                        const int *__restrict__ to,
                                                        const int *__restrict__ from,
                                                        const int *__restrict__ counts)
{
    constexpr uint32_t kSize = TYPE == NUT_F32 ? 4 : 2;
    const uint32_t id = blockIdx.x, c = id % blocks, row = id / blocks;
    const uint32_t h = row % kv.kv_heads, b = row / kv.kv_heads;
    const size_t at = row * history.stride;
    to += size_t(row) * list, from += size_t(row) * list;
    const uint32_t tpr = kv.head_dim / 8, part = threadIdx.x % tpr, group = threadIdx.x / tpr;
    const uint32_t groups = 256 / tpr, column = part * 8 * kSize;
    __shared__ size_t here[256], there[256];
    const uint32_t first = c * 256, r0 = first + threadIdx.x;
    // the list beside its length: what lies behind it is not used
    int dst = r0 < list ? to[r0] : 0, src = r0 < list ? from[r0] : 0;
    const uint32_t total = uint32_t(counts[row]);
    asm volatile("" : "+v"(dst), "+v"(src));
    if (first >= total)
        return;
    const uint32_t count = min(256u, total - first);
    if (r0 < total) {
        const uint32_t to_page = page_of(kv, dst), from_page = page_of(kv, src);
        const float w = history.weights[at + src];
        const int p = history.positions[at + src];
        const size_t x = paged_row(kv, s, b, to_page, dst - to_page * kv.page_size, h);
        const size_t y = paged_row(kv, s, b, from_page, src - from_page * kv.page_size, h);
        history.weights[at + dst] = w;
        history.positions[at + dst] = p;
        here[threadIdx.x] = y == kNoRow ? kNoRow : x;
        there[threadIdx.x] = x == kNoRow ? kNoRow : y;
    }
    __syncthreads();
    if (group >= groups)
        return;
    typedef uint32_t Piece __attribute__((ext_vector_type(4)));
    constexpr int kPieces = kSize / 2, kRows = 4; // rows in flight
    for (uint32_t r = group; r < count; r += kRows * groups) {
        Piece k[kRows][kPieces], v[kRows][kPieces];
#pragma unroll
        for (int i = 0; i < kRows; i++) {
            const size_t y = there[min(r + i * groups, count - 1)];
            const size_t from_row = y == kNoRow ? 0 : y;
#pragma unroll
            for (int w = 0; w < kPieces; w++) {
                k[i][w] = reinterpret_cast<const Piece *>(kv.keys + from_row + column)[w];
                v[i][w] = reinterpret_cast<const Piece *>(kv.values + from_row + column)[w];
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; i++) {
            const size_t x = r + i * groups < count ? here[r + i * groups] : kNoRow;
            if (x != kNoRow)
#pragma unroll
                for (int w = 0; w < kPieces; w++) {
                    reinterpret_cast<Piece *>(kv.keys + x + column)[w] = k[i][w];
                    reinterpret_cast<Piece *>(kv.values + x + column)[w] = v[i][w];
                }
        }
    }
    if (kv.bounds == nullptr)
        return;
    // head_dim / 8 threads a page: the list is in the order of rows, so a page's
    // entries are a run of it
    for (uint32_t r = group; r < count; r += groups) {
        const uint32_t page = page_of(kv, to[first + r]);
        if (first + r != 0 && page_of(kv, to[first + r - 1]) == page)
            continue; // not its first
        if (paged_row(kv, s, b, page, 0, h) == kNoRow)
            continue;
        char *bounds = kv.bounds + (size_t(s.table[size_t(b) * s.table_stride + page]) *
                                        kv.kv_heads + h) * 2 * kv.head_dim * kSize + column;
        float lo[8], hi[8];
        load8<TYPE>(bounds, lo);
        load8<TYPE>(bounds + kv.head_dim * kSize, hi);
        for (uint32_t e = first + r; e < total && page_of(kv, to[e]) == page; e++) {
            const uint32_t from_page = page_of(kv, from[e]);
            const size_t y = paged_row(kv, s, b, from_page, from[e] - from_page * kv.page_size, h);
            if (y == kNoRow)
                continue;
            float x[8];
            load8<TYPE>(kv.keys + y + column, x);
#pragma unroll
            for (int j = 0; j < 8; j++)
                lo[j] = lower(lo[j], x[j]), hi[j] = upper(hi[j], x[j]);
        }
        store8<TYPE>(bounds, lo);
        store8<TYPE>(bounds + kv.head_dim * kSize, hi);
    }
}

uint32_t pages_of(const PagedView &kv, uint32_t rows) { return page_of(kv, rows - 1) + 1; }

size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

template <int TYPE, int GH, uint32_t LANES>
void scores_by(const PagedView &kv, const PagedSeqs &seqs, const float *query,
               size_t query_stride, uint32_t heads, uint64_t *scores, hipStream_t stream)
{
    const uint32_t width = pages_of(kv, seqs.max_length), per_block = 256 / LANES;
    const uint32_t blocks = (width + per_block - 1) / per_block;
    hipLaunchKernelGGL((page_scores_kernel<TYPE, GH, LANES>),
                       paged_grid(uint64_t(seqs.batch) * kv.kv_heads * blocks, 256), dim3(256), 0,
                       stream, kv, seqs, query, query_stride, heads, blocks, width, scores);
}

template <int TYPE, int GH>
void scores_of(const PagedView &kv, const PagedSeqs &seqs, const float *query,
               size_t query_stride, uint32_t heads, uint64_t *scores, hipStream_t stream)
{
    const auto run = kv.head_dim <= 32    ? scores_by<TYPE, GH, 4>
                     : kv.head_dim <= 64  ? scores_by<TYPE, GH, 8>
                     : kv.head_dim <= 128 ? scores_by<TYPE, GH, 16>
                                          : scores_by<TYPE, GH, 32>;
    run(kv, seqs, query, query_stride, heads, scores, stream);
}

template <int TYPE>
void scores_mfma(const PagedView &kv, const PagedSeqs &seqs, const float *query,
                 size_t query_stride, uint32_t heads, uint64_t *scores, hipStream_t stream)
{
    const uint32_t width = pages_of(kv, seqs.max_length), blocks = (width + 63) / 64;
    hipLaunchKernelGGL(page_scores_mfma_kernel<TYPE>,
                       paged_grid(uint64_t(seqs.batch) * kv.kv_heads * blocks, 256), dim3(256), 0,
                       stream, kv, seqs, query, query_stride, heads, blocks, width, scores);
}

template <int TYPE>
void scores_for(const PagedView &kv, const PagedSeqs &seqs, const float *query,
                size_t query_stride, uint32_t heads, uint64_t *scores, hipStream_t stream)
{
    // The matrix instruction's 16 columns are worth it from five heads on. Both
    // calls of a selection, us with its own kernel and with the matrix one: one
    // head of 128, 4 sequences of 16,000 rows 15.5 and 27.7; two heads 10.4 and
    // 12.4; four 10.7 and 12.2; eight (four at a time) 14.1 and 11.4.
    const uint32_t group = heads / kv.kv_heads;
    const auto run = group == 1   ? scores_of<TYPE, 1>
                     : group == 2 ? scores_of<TYPE, 2>
                     : group <= 4 ? scores_of<TYPE, 4>
                                  : scores_mfma<TYPE>;
    run(kv, seqs, query, query_stride, heads, scores, stream);
}

} // namespace

void launch_paged_append(const PagedView &kv, const PagedSeqs &seqs, const float *keys,
                         const float *values, size_t rows, size_t row_stride,
                         size_t head_stride, const int *starts, uint32_t each,
                         uint32_t max_new, const PagedHistory &history, const int *firsts,
                         int *new_lengths, hipStream_t stream)
{
    const uint32_t touched = pages_touched(max_new, kv.page_size);
    const uint32_t threads = append_threads(kv.page_size, max_new, kv.head_dim);
    const auto kernel = kv.type == NUT_F32   ? append_kernel<NUT_F32>
                        : kv.type == NUT_F16 ? append_kernel<NUT_F16>
                                             : append_kernel<NUT_BF16>;
    hipLaunchKernelGGL(kernel, paged_grid(uint64_t(seqs.batch) * kv.kv_heads * touched, threads),
                       dim3(threads), 0, stream, kv, seqs, keys, values, rows, row_stride,
                       head_stride, starts, each, max_new, history, firsts, new_lengths, touched);
    check_launch("paged append");
}

size_t select_workspace(const PagedView &kv, const PagedSeqs &seqs)
{
    paged_grid(uint64_t(seqs.batch) * kv.kv_heads, 256);
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
    // sequences of no more than `top` pages read them all
    if (pages_of(kv, seqs.max_length) > top) {
        run(kv, seqs, query, query_stride, heads, scores, stream);
        check_launch("paged select");
    }
    hipLaunchKernelGGL(choose_pages_kernel, paged_grid(uint64_t(seqs.batch) * kv.kv_heads, 256),
                       dim3(256), 0, stream, kv, seqs, scores, pages_of(kv, seqs.max_length), top, first, last,
                       selected);
    check_launch("paged select");
}

// Rows of a sequence and KV head that move at most: into the budget's places,
// from behind them.
static uint32_t most_moved(const PagedSeqs &seqs, uint32_t budget)
{
    return budget < seqs.max_length ? std::min(budget, seqs.max_length - budget) : 0;
}

// Workgroups that move the rows of a list.
static uint32_t move_blocks(uint32_t list) { return (list + 255) / 256; }

size_t evict_workspace(const PagedView &kv, const PagedSeqs &seqs, uint32_t budget)
{
    const size_t heads = size_t(seqs.batch) * kv.kv_heads;
    paged_grid(heads, 1024);
    paged_grid(heads * move_blocks(most_moved(seqs, budget)), 256);
    return 2 * aligned(heads * most_moved(seqs, budget) * sizeof(int)) +
           aligned(heads * sizeof(int));
}

void launch_paged_evict(const PagedView &kv, const PagedSeqs &seqs, const PagedHistory &history,
                        uint32_t budget, uint32_t first, uint32_t last, int *new_lengths,
                        char *workspace, hipStream_t stream)
{
    const uint64_t heads = uint64_t(seqs.batch) * kv.kv_heads;
    const uint32_t list = most_moved(seqs, budget);
    const size_t bytes = aligned(heads * list * sizeof(int));
    int *to = reinterpret_cast<int *>(workspace);
    int *from = reinterpret_cast<int *>(workspace + bytes);
    int *counts = reinterpret_cast<int *>(workspace + 2 * bytes);
    // eight rows a thread of the smaller workgroup
    const uint32_t threads = seqs.max_length <= 2048 ? 256 : 1024;
    hipLaunchKernelGGL(threads == 256 ? plan_eviction_kernel<256> : plan_eviction_kernel<1024>,
                       paged_grid(heads, threads), dim3(threads), 0, stream, kv, seqs, history,
                       budget, first, last, list, new_lengths, to, from, counts);
    check_launch("paged evict");
    if (list == 0)
        return;
    const uint32_t blocks = move_blocks(list);
    const auto kernel = kv.type == NUT_F32   ? move_rows_kernel<NUT_F32>
                        : kv.type == NUT_F16 ? move_rows_kernel<NUT_F16>
                                             : move_rows_kernel<NUT_BF16>;
    hipLaunchKernelGGL(kernel, paged_grid(heads * blocks, 256), dim3(256), 0, stream, kv, seqs,
                       history, list, blocks, to, from, counts);
    check_launch("paged evict");
}

} // namespace nut
