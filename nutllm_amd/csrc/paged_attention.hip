// paged_attention.hip — attention of one new token a sequence over a paged
// KV cache.
//
// A workgroup takes a run of one sequence's rows for one KV head and up to 16
// of the query heads that share it, and reads each row once. Its waves, four
// at most, take tiles of the run in turn, each with a softmax of its own
// (running maximum and sum); they are joined at the end, and the runs by
// join_kernel.
//
// Everything between a tile's loads and its products stays in the lane that
// it was loaded into. With lane = 16 j + c, the matrix instruction for
// S = K Q^T (rows: keys, columns: heads) takes row c's components from lane
// (j, c) and leaves the scores of keys 4 j + i (i = 0..3) and head c there.
// The one for O^T = V^T P^T sums over keys in an order of our choice, so lane
// (j, c) supplies exactly those keys: P needs no exchange, and lane (j, c)
// loads V rows 4 j + i, in pieces of E components (up to 16 bytes) that lie
// beside the other lanes', from 16 E w + E c on for w = 0, 1, ..: the t-th
// component that it holds is row c of output tile t. With a lane's pieces one
// after another instead, loads ask for lines by halves: 24 sequences of 6,000
// fp32 rows of 96, 128 components 172, 218 us for 153, 196. Only the running
// maximum crosses lanes.
//
// fp32 rows run on v_mfma_f32_16x16x4f32; 16-bit rows on the 16x16x32 forms,
// with the fp32 operand (the query, the weights) split into limbs of the rows'
// type, whose products with a row are exact. Three bfloat16 limbs of 8 bits are
// all 24 bits of it. Two fp16 limbs are 23, a rounding of 2^-23 of a component's
// size, down to fp16's smallest step: the query is scaled by a power of two so
// that its largest component lies in [2^13, 2^14), and weights lie in [0, 2^14],
// so that what is left out of a query's component is at most 2^-38 of the
// largest one besides, of a weight 2^-39 of the largest. That shows in
// components 2^15 and more below the largest, and in scores only where a row is
// near zero in the large ones; a third limb would not reach lower, and cost
// half as many products again. Accumulation is fp32.
//
// HBM bounds long calls: 2.0 GB of fp16 rows (4 sequences of up to 32,768, 32
// heads of 128) in 304 us, 6.4 TB/s. 32 sequences of up to 2,048 bfloat16 rows
// (34 MB) take 13.5 us, of which two launches are 8.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "paged_attend.hpp"
#include "runtime.hpp"

namespace nut {

namespace {

constexpr uint32_t kMostRows = 1024; // of a run

struct AttendArgs {
    PagedView kv;
    PagedSeqs s;
    const float *query;
    size_t query_stride;
    uint32_t heads, group;
    float scale; // times log2(e)
    const int *selected;
    uint32_t top;
    float *out, *lse;
    uint32_t chunk, chunks, tiles;
    uint32_t turn; // runs begin one further every 2^turn heads
    // A selection of more pages than a sequence has: runs without any end early,
    // which costs the others a barrier (64 pages of 128 rows, 33 sequences of up
    // to 537 rows, 32 KV heads of 128: 83 us with it and 115 without; where no run
    // is empty, 32 of 501 pages, 18.1 and 17.7).
    bool loose;
    float *parts;  // [batch][heads][chunks][head_dim], unnormalised
    float2 *stats; // [batch][heads][chunks]: exponent they refer to, sum
    float *scores; // [batch][heads][chunks * chunk], base 2; nullptr: not kept
};

// Where a row lies: page `index` of the sequence (-1: none, -2: one that no
// table row has), and what the table says of it.
struct Place {
    int index, page;
    uint32_t slot;
};

// Row i of the run at `begin`, before the table is asked.
__device__ __forceinline__ Place place_of(const AttendArgs &a, uint32_t b, uint32_t h, uint32_t i,
                                          uint32_t begin, uint32_t most, uint32_t pages)
{
    Place p{-1, -1, 0};
    if (i >= a.chunk || begin + i >= most)
        return p;
    p.index = int(page_of(a.kv, begin + i));
    p.slot = begin + i - uint32_t(p.index) * a.kv.page_size;
    if (a.selected != nullptr) {
        p.index = a.selected[(size_t(b) * a.kv.kv_heads + h) * a.top + p.index];
        if (p.index < -1 || p.index >= int(pages))
            p.index = -2;
    }
    return p;
}

// Waves of a workgroup at most: their sums have to fit its 64 KB of shared
// memory. Runs of one or two tiles have a wave a tile: one that only waits
// would keep others' registers (bfloat16 rows at 32 KV heads of 128: 61
// sequences of up to 17 rows 18.6 us with four waves and 7.6 with one, 27 of up
// to 33 10.4 with four and 6.7 with two). The count is the kernel's type: as an
// argument it cost 32 sequences of 2,048 rows 14.7 us for 13.6.
template <int HD> constexpr int kWavesOf = HD == 256 ? 2 : 4;

template <int TYPE, int HD, bool FULL, bool NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void attend_kernel(AttendArgs a)
{
    using T = Tile<TYPE, HD>;
    constexpr int G = T::G, kThreads = 64 * WAVES;
    constexpr int kStride = HD + 4; // of a head's sums: 16 lanes' rows on all banks
    // with fewer waves than there may be, a tile each
    constexpr uint32_t kRoom = WAVES == kWavesOf<HD> ? kMostRows : 64;
    static_assert(WAVES == kWavesOf<HD> || WAVES * T::kRows <= int(kRoom), "rows of a short run");
    // the rows' offsets, and when they are done with the waves' sums
    __shared__ union Shared {
        size_t at[kRoom];
        float o[WAVES][16][kStride];
    } lds;
    __shared__ float stat[3][WAVES][16];
    __shared__ uint32_t gone[kRoom / 32]; // bit per row: masked
    const PagedView &kv = a.kv;
    // A sequence's runs one after another, begun one further every 2^turn: the
    // workgroups go to 8 XCDs in turn, and on each to 4 groups of its CUs. If
    // runs began alike, or moved on where these 32 have not been through, some
    // would get all of the late runs, which short sequences, and selections of
    // few pages, have not (33 sequences of up to 537 fp16 rows, 32 KV heads of
    // 128, in the first of four runs of a selection: 144 us when runs moved on
    // every two heads, 79 every eight).
    const uint32_t b = blockIdx.z, h = a.tiles == 1 ? blockIdx.y : blockIdx.y / a.tiles;
    const uint32_t tile16 = blockIdx.y - h * a.tiles;
    const uint32_t c = (blockIdx.x + ((blockIdx.y + gridDim.y * b) >> a.turn)) % a.chunks;
    const uint32_t begin = c * a.chunk;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int j = lane >> 4, column = lane & 15;
    const uint32_t first = tile16 * 16, here = min(16u, a.group - first);
    const bool valid = uint32_t(column) < here;
    const size_t row = size_t(b) * a.heads + h * a.group + first;
    const size_t mine = row + (valid ? column : 0);
    Query<TYPE, HD> q;
    q.fetch(a.query + b * a.query_stride + (mine - size_t(b) * a.heads) * kv.head_dim, valid,
            kv.head_dim, lane);

    // Where the run's rows begin, so that pages need not fit tiles. The entries
    // of the table are fetched together, and beside the length, not after it:
    // what lies behind the length is not used.
    const uint32_t most = a.selected == nullptr ? a.s.max_length : a.top * kv.page_size;
    const uint32_t pages = page_of(kv, a.s.max_length - 1) + 1;
    constexpr int kEach = (kRoom + kThreads - 1) / kThreads;
    Place places[kEach];
#pragma unroll
    for (int e = 0; e < kEach; e++)
        places[e] = place_of(a, b, h, e * kThreads + threadIdx.x, begin, most, pages);
    if (a.loose) {
        bool some = false;
#pragma unroll
        for (int e = 0; e < kEach; e++)
            some = some || places[e].index != -1;
        if (!__syncthreads_or(some)) { // no row: the join passes it over
            if (c == 0 && h == 0)
                (void)paged_length(kv, a.s, b, threadIdx.x == 0); // but reports a bad length
            if (threadIdx.x < here)
                a.stats[(row + threadIdx.x) * a.chunks + c] = make_float2(-INFINITY, 0.0f);
            return;
        }
    }
#pragma unroll
    for (int e = 0; e < kEach; e++)
        if (places[e].index >= 0)
            places[e].page = a.s.table[size_t(b) * a.s.table_stride + places[e].index];
    const uint32_t n = paged_length(kv, a.s, b, threadIdx.x == 0 && c == 0 && h == 0);
#pragma unroll
    for (int e = 0; e < kEach; e++)
        asm volatile("" : "+v"(places[e].page));
    const uint32_t total = a.selected == nullptr ? n : most;
    if (begin >= total && c != 0)
        return;
    const uint32_t count = min(total - begin, a.chunk);
    const int tiles = int((count + T::kRows - 1) / T::kRows);
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        const uint32_t i = e * kThreads + threadIdx.x;
        if (i >= (count + kWave - 1) / kWave * kWave)
            break;
        const Place place = places[e];
        size_t at = 0;
        bool out = true;
        if (i < count && place.index < -1)
            paged_flag(kv.status, kBadPage);
        if (i < count && place.index >= 0 &&
            uint64_t(place.index) * kv.page_size + place.slot < n) {
            out = !page_in(place.page, kv.pages);
            if (!out)
                at = size_t(place.page) * kv.page_stride + h * kv.head_stride +
                     place.slot * kv.slot_stride;
            else
                paged_flag(kv.status, kBadPage);
        }
        lds.at[i] = at;
        const uint64_t masked = __ballot(out);
        if (lane % 32 == 0)
            gone[i / 32] = uint32_t(masked >> lane);
    }

    float *scores = a.scores != nullptr && valid
                        ? a.scores + mine * a.chunks * a.chunk + begin + 4 * j
                        : nullptr;
    Softmax<TYPE, HD> sm;
    __syncthreads();
    // One tile in registers a wave: in long calls the other waves of the SIMD (four
    // and more up to 64 components) keep loads in flight, and a second tile in
    // registers cost their places: 378 us for 337 where both were measured. Short
    // calls have little more than a wave a SIMD (308 workgroups with rows), and
    // wait for each tile; a second one cost them too (13.2 to 14.4 us).
    Tile<TYPE, HD> x;
    constexpr uint32_t kAll = T::kWide ? 0xffffu : 0xffffffffu;
    const auto masked = [&](int t) {
        return uint32_t(__builtin_amdgcn_readfirstlane(
            gone[t * T::kRows / 32] >> (t * T::kRows % 32) & kAll));
    };
    // the wave's next tile; of a selection, which may hold fewer pages than there
    // is room for, the next one that has a row
    const auto next = [&](int t) {
        while (a.selected != nullptr && t < tiles && masked(t) == kAll)
            t += WAVES;
        return t;
    };
    int t = next(wave);
    if (t < tiles)
        x.template load<FULL, NT>(kv, lds.at + t * T::kRows, lane);
    q.convert(a.scale);
    while (t < tiles) {
        attend<TYPE, HD>(x, masked(t), q, sm, scores == nullptr ? nullptr : scores + t * T::kRows,
                         lane);
        t = next(t + WAVES);
        if (t < tiles)
            x.template load<FULL, NT>(kv, lds.at + t * T::kRows, lane);
    }
    sm.sum += __shfl_xor(sm.sum, 16);
    sm.sum += __shfl_xor(sm.sum, 32);

    // The waves' sums side by side; then a thread per four components adds them.
    __syncthreads();
    if (j == 0)
        stat[0][wave][column] = sm.most, stat[1][wave][column] = sm.ref,
        stat[2][wave][column] = sm.sum;
    {
        constexpr int E = T::kEach;
#pragma unroll
        for (int p = 0; p < G; p += E) {
            float flat[4 * E]; // components 16 p + 4 j E .. of the lane's head
#pragma unroll
            for (int t = 0; t < E; t++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    flat[i * E + t] = sm.o[p + t][i];
            float *to = lds.o[wave][column] + 16 * p + 4 * j * E;
#pragma unroll
            for (int d = 0; d < 4 * E; d += 4)
                *reinterpret_cast<f32x4 *>(to + d) =
                    f32x4{flat[d], flat[d + 1], flat[d + 2], flat[d + 3]};
        }
    }
    __syncthreads();
    const uint32_t parts = FULL ? HD / 4 : kv.head_dim / 4;
    for (uint32_t i = threadIdx.x; i < here * parts; i += kThreads) {
        const uint32_t head = i / parts, d = i % parts * 4;
        float most = stat[0][0][head];
#pragma unroll
        for (int w = 1; w < WAVES; w++)
            most = fmaxf(most, stat[0][w][head]);
        const float ref = most == -INFINITY ? 0.0f : most - Softmax<TYPE, HD>::kShift;
        float sum = 0.0f;
        f32x4 o{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            // what no row of a finite score reached is zero, or not a number
            const float f = stat[0][w][head] == -INFINITY
                                ? 1.0f
                                : __builtin_amdgcn_exp2f(stat[1][w][head] - ref);
            sum = fmaf(stat[2][w][head], f, sum);
            const f32x4 y = *reinterpret_cast<const f32x4 *>(&lds.o[w][head][d]);
#pragma unroll
            for (int e = 0; e < 4; e++)
                o[e] = fmaf(y[e], f, o[e]);
        }
        const size_t at = row + head;
        if (a.parts != nullptr) {
            *reinterpret_cast<f32x4 *>(a.parts + (at * a.chunks + c) * kv.head_dim + d) = o;
            if (d == 0)
                a.stats[at * a.chunks + c] = make_float2(sum == 0.0f ? -INFINITY : ref, sum);
        } else {
            // no weight: zeros, whatever the values are
            *reinterpret_cast<f32x4 *>(a.out + at * kv.head_dim + d) =
                sum == 0.0f ? f32x4{0, 0, 0, 0} : o * (1.0f / sum);
            if (d == 0 && a.lse != nullptr)
                a.lse[at] = sum == 0.0f ? -INFINITY : (ref + log2f(sum)) * 0.69314718055994531f;
        }
    }
}

// One head's runs joined: tpr = head_dim / 4 threads hold four components each,
// and the workgroup's groups of tpr threads take runs in turn. The first
// run of a group is fetched beside the length, before it is known to count.
__device__ __forceinline__ void join_head(const AttendArgs &a, uint32_t row, float *red,
                                          f32x4 *acc)
{
    const PagedView &kv = a.kv;
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const uint32_t waves = blockDim.x / kWave, tpr = kv.head_dim / 4;
    const uint32_t part = threadIdx.x % tpr, g = threadIdx.x / tpr, groups = blockDim.x / tpr;
    const float2 *stats = a.stats + size_t(row) * a.chunks;
    const f32x4 *parts =
        reinterpret_cast<const f32x4 *>(a.parts + size_t(row) * a.chunks * kv.head_dim) + part;
    float2 own{-INFINITY, 0.0f};
    if (threadIdx.x < a.chunks)
        own = stats[threadIdx.x];
    f32x4 ahead{0, 0, 0, 0};
    if (g < groups && g < a.chunks)
        ahead = parts[g * tpr];
    const uint32_t n = paged_length(kv, a.s, row / a.heads, false);
    asm volatile("" : "+v"(own.x), "+v"(own.y), "+v"(ahead));
    const uint32_t total = a.selected == nullptr ? n : a.top * kv.page_size;
    const uint32_t runs = (total + a.chunk - 1) / a.chunk;

    // Runs that no row of a finite score reached hold ref = -inf: their sums
    // are not read.
    float most = threadIdx.x < runs ? own.x : -INFINITY;
    for (uint32_t i = threadIdx.x + blockDim.x; i < runs; i += blockDim.x)
        most = fmaxf(most, stats[i].x);
    most = wave_max(most);
    if (waves > 1) {
        if (lane == 0)
            red[wave] = most;
        __syncthreads();
        for (uint32_t w = 0; w < waves; w++)
            most = fmaxf(most, red[w]);
    }
    float sum = 0.0f;
    f32x4 o{0, 0, 0, 0};
    if (g < groups)
        for (uint32_t i = g; i < runs; i += groups) {
            const float2 st = stats[i];
            const f32x4 x = i == g ? ahead : parts[i * tpr];
            if (st.x == -INFINITY)
                continue;
            const float f = __builtin_amdgcn_exp2f(st.x - most);
            sum = fmaf(st.y, f, sum);
#pragma unroll
            for (int e = 0; e < 4; e++)
                o[e] = fmaf(x[e], f, o[e]);
        }
    acc[2 * threadIdx.x] = o;
    acc[2 * threadIdx.x + 1][0] = sum;
    __syncthreads();
    if (g != 0)
        return;
    for (uint32_t i = 1; i < groups; i++) {
        o += acc[2 * (i * tpr + part)];
        sum += acc[2 * (i * tpr + part) + 1][0];
    }
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    *reinterpret_cast<f32x4 *>(a.out + size_t(row) * kv.head_dim + part * 4) = o * f;
    if (part == 0 && a.lse != nullptr)
        a.lse[row] = sum == 0.0f ? -INFINITY : (most + log2f(sum)) * 0.69314718055994531f;
}

// The weights of four rows a thread, over the heads that share them, 8 at a
// time: 8 lanes a head find its maximum and sum from the runs, while the
// scores are on their way.
__device__ __forceinline__ void weigh_rows(const AttendArgs &a, const PagedHistory &history,
                                           uint32_t b, uint32_t h, uint32_t first, float *base)
{
    constexpr int kHeads = 8;
    const PagedView &kv = a.kv;
    const uint32_t n = paged_length(kv, a.s, b, false);
    if (first >= n)
        return;
    const uint32_t runs = (n + a.chunk - 1) / a.chunk, span = a.chunks * a.chunk;
    float grown[4] = {0, 0, 0, 0};
    for (uint32_t g = 0; g < a.group; g += kHeads) {
        const uint32_t here = min(uint32_t(kHeads), a.group - g);
        const size_t row = size_t(b) * a.heads + h * a.group + g;
        float s[kHeads][4];
#pragma unroll
        for (int k = 0; k < kHeads; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t i = first + e * blockDim.x + threadIdx.x;
                s[k][e] = uint32_t(k) < here && i < n ? a.scores[(row + k) * span + i] : -INFINITY;
            }
        __syncthreads();
        for (uint32_t k = threadIdx.x / 8; k < here; k += blockDim.x / 8) {
            float most = -INFINITY, sum = 0.0f;
            for (uint32_t i = threadIdx.x % 8; i < runs; i += 8) {
                const float2 st = a.stats[(row + k) * a.chunks + i];
                if (st.x == -INFINITY)
                    continue;
                const float now = fmaxf(most, st.x);
                sum = sum * __builtin_amdgcn_exp2f(most - now) +
                      st.y * __builtin_amdgcn_exp2f(st.x - now);
                most = now;
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                const float m = __shfl_xor(most, o), z = __shfl_xor(sum, o);
                const float now = fmaxf(most, m);
                if (now != -INFINITY)
                    sum = (most == -INFINITY ? 0.0f : sum * __builtin_amdgcn_exp2f(most - now)) +
                          (m == -INFINITY ? 0.0f : z * __builtin_amdgcn_exp2f(m - now));
                most = now;
            }
            // no weight where nothing has any
            if (threadIdx.x % 8 == 0)
                base[k] = most == -INFINITY ? INFINITY : most + log2f(sum);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kHeads; k++)
            if (uint32_t(k) < here)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    grown[e] += __builtin_amdgcn_exp2f(s[k][e] - base[k]);
    }
    float *weights = history.weights + (size_t(b) * kv.kv_heads + h) * history.stride;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const uint32_t i = first + e * blockDim.x + threadIdx.x;
        if (i < n)
            weights[i] += grown[e];
    }
}

// One launch for both: 3 us of 32 x 32 heads of four runs, 5.6 us with the
// weights of 16 sequences of up to 4,096 rows. The first batch x heads
// workgroups join a head's runs; the others, `blocks`
// for each sequence and KV head, add the weights of 4 rows a thread.
__global__ __launch_bounds__(256) void join_kernel(AttendArgs a, PagedHistory history,
                                                   uint32_t joins, uint32_t blocks)
{
    __shared__ float red[8];
    __shared__ f32x4 acc[512];
    if (blockIdx.x < joins) {
        join_head(a, blockIdx.x, red, acc);
    } else {
        const uint32_t id = blockIdx.x - joins, h = id / blocks % a.kv.kv_heads;
        weigh_rows(a, history, id / blocks / a.kv.kv_heads, h, id % blocks * 4 * blockDim.x, red);
    }
}

// Rows beyond this many bytes go past the caches' replacement: nothing of them
// is there when the next call comes, and HBM is read faster without it. Three
// caches in turn, us a call without and with, by MB of a call's rows: bfloat16
// 33 15.3 16.3, 66 19.8 21.7, 131 33.3 30.6, 524 108 96, fp16 131 32.9 33.4, 262
// 54 52, 2,097 359 328, fp32 131 32 30, 2,097 372 334. Not where sixteen pieces
// are less than a line, nor of rows shorter than HD, whose lines' ends would be
// fetched again: 16-bit rows of 96 components 86 without and 92 with (orders of
// slots first 95 and 112), fp32 rows of 80 52 and 55.
constexpr uint64_t kPastCaches = 128ull << 20;

template <int TYPE, int HD, bool FULL, bool NT, int WAVES>
void attend_by(const AttendArgs &a, dim3 grid, hipStream_t stream)
{
    hipLaunchKernelGGL((attend_kernel<TYPE, HD, FULL, NT, WAVES>), grid, dim3(64 * WAVES), 0,
                       stream, a);
}

template <int TYPE, int HD>
void attend_as(const AttendArgs &a, dim3 grid, uint32_t rows, uint64_t bytes, hipStream_t stream)
{
    constexpr int kMost = kWavesOf<HD>;
    const bool full = a.kv.head_dim == HD;
    const uint32_t tiles = (std::min(a.chunk, rows) - 1) / Tile<TYPE, HD>::kRows + 1;
    auto run = tiles == 1   ? (full ? attend_by<TYPE, HD, true, false, 1>
                                    : attend_by<TYPE, HD, false, false, 1>)
               : tiles == 2 ? (full ? attend_by<TYPE, HD, true, false, 2>
                                    : attend_by<TYPE, HD, false, false, 2>)
                            : (full ? attend_by<TYPE, HD, true, false, kMost>
                                    : attend_by<TYPE, HD, false, false, kMost>);
    if constexpr (Tile<TYPE, HD>::kPiece >= 2)
        if (full && bytes >= kPastCaches)
            run = attend_by<TYPE, HD, true, true, kMost>;
    run(a, grid, stream);
}

template <int TYPE>
void attend_in(const AttendArgs &a, dim3 grid, uint32_t rows, uint64_t bytes, hipStream_t stream)
{
    if (a.kv.head_dim <= 32)
        attend_as<TYPE, 32>(a, grid, rows, bytes, stream);
    else if (a.kv.head_dim <= 64)
        attend_as<TYPE, 64>(a, grid, rows, bytes, stream);
    else if (a.kv.head_dim <= 96)
        attend_as<TYPE, 96>(a, grid, rows, bytes, stream);
    else if (a.kv.head_dim <= 128)
        attend_as<TYPE, 128>(a, grid, rows, bytes, stream);
    else
        attend_as<TYPE, 256>(a, grid, rows, bytes, stream);
}

} // namespace

AttentionPlan plan_attention(const PagedView &kv, const PagedSeqs &seqs, uint32_t heads,
                             uint32_t top, bool weighted)
{
    const auto aligned = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
    AttentionPlan plan{};
    const uint32_t group = heads / kv.kv_heads;
    const uint32_t rows = top == 0 ? seqs.max_length : top * kv.page_size;
    // a selection of more pages than a sequence has is -1 behind them, and tiles
    // without a row are passed over
    const uint32_t likely = plan.likely = std::min(rows, seqs.max_length);
    plan.tiles = (group + 15) / 16;
    // Runs as long as make 512 workgroups, or down to 128 rows, by the longest
    // length (shorter sequences leave some without rows: 308 of 512 have any in
    // the first of these): 32 ragged sequences of up to 2,048 bfloat16 rows, four
    // KV heads, 13.2 us in runs of 512 (512 workgroups), 14.1 in runs of 256 and
    // 15.6 in runs of 1,024; 7 of up to 5,001 fp32 rows, three KV heads, 19.6 in
    // runs of 256 (420 workgroups, 252 with rows) and of 128 (840 and 501), 21.1
    // in runs of 512. A selection of 124 pages of 128 rows from 1,149 fp32 rows:
    // 33 us by the rows that there are, 64 by the places.
    plan.chunk = kMostRows;
    const uint64_t columns = uint64_t(seqs.batch) * kv.kv_heads * plan.tiles;
    while (likely > 128 && plan.chunk > 128 &&
           columns * ((likely + plan.chunk - 1) / plan.chunk) < 512)
        plan.chunk /= 2;
    // Keys of up to 64 KB are one run whatever the number of workgroups: the
    // join's launch costs more. One sequence of 64 components, one run and
    // split: 256 fp32 rows 6.9 and 8.6 us, 512 10.3 and 8.6; 512 bfloat16 rows
    // 7.2 and 8.4, 1,000 10.6 and 8.5.
    if (rows <= kMostRows && uint64_t(likely) * kv.head_dim * paged_element(kv.type) <= 65536)
        plan.chunk = (rows + 127) / 128 * 128;
    plan.chunks = (rows + plan.chunk - 1) / plan.chunk;
    require(seqs.batch <= 65535 && uint64_t(kv.kv_heads) * plan.tiles <= 65535, NUT_EINVAL,
            "paged cache: more rows than one launch covers");
    paged_grid(uint64_t(seqs.batch) * kv.kv_heads * plan.tiles * plan.chunks, 256);
    if (plan.chunks == 1 && !weighted)
        return plan;
    // a wave joins up to 16 runs of a head
    plan.join_threads = plan.chunks <= 16 ? 64 : 256;
    plan.weigh_blocks = weighted ? (seqs.max_length - 1) / (4 * plan.join_threads) + 1 : 0;
    paged_grid(uint64_t(seqs.batch) * (heads + uint64_t(kv.kv_heads) * plan.weigh_blocks),
               plan.join_threads);
    const size_t runs = size_t(seqs.batch) * heads * plan.chunks;
    plan.stats = aligned(runs * kv.head_dim * sizeof(float));
    plan.scores = plan.stats + aligned(runs * sizeof(float2));
    plan.bytes = plan.scores + (weighted ? aligned(runs * plan.chunk * sizeof(float)) : 0);
    return plan;
}

void launch_paged_attention(const PagedView &kv, const PagedSeqs &seqs, const float *query,
                            size_t query_stride, uint32_t heads, float scale,
                            const int *selected, uint32_t top, const PagedHistory &history,
                            float *out, float *lse, char *workspace, hipStream_t stream)
{
    const bool weighted = history.weights != nullptr;
    const AttentionPlan plan = plan_attention(kv, seqs, heads, top, weighted);
    const bool split = plan.bytes != 0;
    AttendArgs a{kv, seqs, query, query_stride, heads, heads / kv.kv_heads,
                 scale * 1.4426950408889634f, selected, top, out, lse, plan.chunk, plan.chunks,
                 plan.tiles, 5 - std::min(5u, uint32_t(__builtin_ctz(plan.chunks))), false, nullptr,
                 nullptr, nullptr};
    if (split) {
        a.loose = top > page_of(kv, seqs.max_length - 1) + 1;
        a.parts = reinterpret_cast<float *>(workspace);
        a.stats = reinterpret_cast<float2 *>(workspace + plan.stats);
        a.scores = weighted ? reinterpret_cast<float *>(workspace + plan.scores) : nullptr;
    }
    const dim3 grid(plan.chunks, kv.kv_heads * plan.tiles, seqs.batch);
    const uint32_t rows = top == 0 ? seqs.max_length : top * kv.page_size;
    const uint64_t bytes = uint64_t(plan.likely) * seqs.batch * kv.kv_heads * kv.head_dim * 2 *
                           paged_element(kv.type);
    if (kv.type == NUT_F32)
        attend_in<NUT_F32>(a, grid, rows, bytes, stream);
    else if (kv.type == NUT_F16)
        attend_in<NUT_F16>(a, grid, rows, bytes, stream);
    else
        attend_in<NUT_BF16>(a, grid, rows, bytes, stream);
    check_launch("paged attention");
    if (!split)
        return;
    const uint32_t joins = seqs.batch * heads;
    hipLaunchKernelGGL(join_kernel, dim3(joins + seqs.batch * kv.kv_heads * plan.weigh_blocks),
                       dim3(plan.join_threads), 0, stream, a, history, joins, plan.weigh_blocks);
    check_launch("paged attention");
}

} // namespace nut
