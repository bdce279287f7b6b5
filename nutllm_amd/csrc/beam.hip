// beam.hip — beam search: the best continuations of every request's beams, and
// the state that goes with them.
//
// Two launches. In the first a wave takes a part of a beam's logits into
// registers: their largest, the sum of their exponentials, and the K largest in
// order. In the second a workgroup per request joins a beam's parts to its
// log-sum, and the beams' lists to the request's K best. Only the logits' order
// matters within a beam, so that ranks are worked out for few candidates, in 64 bits.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "device.hpp"
#include "paged_device.hpp"
#include "runtime.hpp"
#include "serving.hpp"

namespace nut {

namespace {

constexpr uint32_t kMostParts = 64;   // of a beam's logits: a lane each
constexpr int kFound = 64;           // keys that a wave ranks at once
constexpr uint32_t kMostListed = 2048; // keys of a beam's parts: 32 parts of 64
constexpr int kChosen = 512;         // candidates of a request that are ranked at once

struct Part {
    float most; // minus infinity: no finite one
    uint32_t unused;
    double sum; // of exp(logit - most); not a number after one that is none
};

struct BeamArgs {
    BeamsView from, to;
    const void *logits;
    size_t row_stride;
    uint32_t vocab, parts;
    int eos;
    float power;
    int *parents, *tokens;
    Part *stats;    // [requests][beams][parts]
    uint64_t *best; // [requests][beams][parts][to.beams]: keys in descending order, then 0
};

// An order of 64-bit keys: the larger logit, then the lower token. 0: none.
__device__ __forceinline__ uint64_t key_of(float v, uint32_t token)
{
    const uint32_t u = __float_as_uint(v + 0.0f); // -0 is 0
    const uint32_t order = u & 0x80000000u ? ~u : u | 0x80000000u;
    return uint64_t(order) << 32 | uint32_t(~token);
}
__device__ __forceinline__ float logit_of(uint64_t key)
{
    const uint32_t order = uint32_t(key >> 32);
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint32_t token_of(uint64_t key) { return ~uint32_t(key); }

// Ranks as keys in the same order; 0 for minus infinity and what is no number.
__device__ __forceinline__ uint64_t rank_key(double v)
{
    if (!(v > -INFINITY))
        return 0;
    const uint64_t u = uint64_t(__double_as_longlong(v + 0.0));
    return u >> 63 ? ~u : u | (uint64_t(1) << 63);
}

template <int CTRL, int ROWS = 0xF> __device__ __forceinline__ uint32_t dpp_max(uint32_t v)
{
    return max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, ROWS, 0xF, false)));
}

// The largest of a wave's values, in every lane: 12 moves within the registers, the
// upper halves first (through shared memory 64-bit values took 600 cycles).
__device__ __forceinline__ uint32_t wave_most(uint32_t v)
{
    v = dpp_max<kDppQuadSwap1>(v);
    v = dpp_max<kDppQuadSwap2>(v);
    v = dpp_max<kDppRowHalfMirror>(v);
    v = dpp_max<kDppRowMirror>(v);
    v = dpp_max<kDppRowBcast15, 0xA>(v);
    v = dpp_max<kDppRowBcast31, 0xC>(v);
    return uint32_t(__builtin_amdgcn_readlane(int(v), 63));
}
__device__ __forceinline__ uint64_t wave_most(uint64_t v)
{
    const uint32_t hi = wave_most(uint32_t(v >> 32));
    return uint64_t(hi) << 32 | wave_most(uint32_t(v >> 32) == hi ? uint32_t(v) : 0u);
}

// A lane's value, the same for all.
__device__ __forceinline__ uint64_t lane_of(uint64_t v, uint32_t lane)
{
    return uint64_t(uint32_t(__builtin_amdgcn_readlane(int(v >> 32), lane))) << 32 |
           uint32_t(__builtin_amdgcn_readlane(int(v), lane));
}

// What the wave's lanes wrote to shared memory, its other lanes read.
__device__ __forceinline__ void wave_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// exp(d), d <= 0: the exponent in base 2 in two pieces, so that the error is
// that of the instruction, a unit in the last place, however large d is.
__device__ __forceinline__ float exp_below(float d)
{
    const float t = d * 1.44269504f;
    const float rest = fmaf(d, 1.92596299e-8f, fmaf(d, 1.44269504f, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, rest * 0.69314718f, e);
}

// 16 bytes of a row, which may begin at any element.
template <int TYPE> struct __attribute__((packed, aligned(TYPE == NUT_F32 ? 4 : 2))) Run {
    uint32_t w[4];
};

// EACH logits a lane, in runs of 16 bytes: run r of the wave's part is lane r % 64's.
// 512 beams of 100,003 fp16 logits: 37 us, 2.7 TB/s; exponentials and the search bound it
// (with the bound searched among 64-bit keys, and a pass of its own for what is no number,
// 47; with every key found by a reduction of its own 84).
template <int TYPE, int EACH>
__global__ __launch_bounds__(kWave) void scan_kernel(BeamArgs a)
{
    constexpr int kRun = TYPE == NUT_F32 ? 4 : 8, kRuns = EACH / kRun;
    constexpr uint32_t kPart = kWave * EACH;
    const uint32_t lane = threadIdx.x, part = blockIdx.x, row = blockIdx.y + gridDim.y * blockIdx.z;
    if (row >= a.from.requests * a.from.beams)
        return;
    if (!(a.from.scores[row] > -INFINITY) || (a.from.ended != nullptr && a.from.ended[row] != 0))
        return; // no beam, or one that needs no logits
    constexpr int kSize = TYPE == NUT_F32 ? 4 : 2;
    const char *logits = static_cast<const char *>(a.logits) + row * a.row_stride * kSize;
    // Runs by token, not by address: beams with the same logits have the same sums,
    // to the last bit, wherever their rows begin.
    float v[EACH];
#pragma unroll
    for (int r = 0; r < kRuns; r++) {
        const uint32_t at = part * kPart + (r * kWave + lane) * kRun;
        if (at + kRun <= a.vocab) {
            const Run<TYPE> x = *reinterpret_cast<const Run<TYPE> *>(logits + size_t(at) * kSize);
#pragma unroll
            for (int e = 0; e < kRun; e++)
                v[r * kRun + e] = TYPE == NUT_F32 ? __uint_as_float(x.w[e % 4])
                                  : TYPE == NUT_BF16
                                      ? from_bf16(x.w[e / 2 % 4] >> (e % 2 * 16) & 0xffffu)
                                      : from_f16(x.w[e / 2 % 4] >> (e % 2 * 16) & 0xffffu);
        } else {
#pragma unroll
            for (int e = 0; e < kRun; e++) {
                float x = -INFINITY;
                if (at + e < a.vocab) {
                    const char *p = logits + size_t(at + e) * kSize;
                    x = TYPE == NUT_F32    ? *reinterpret_cast<const float *>(p)
                        : TYPE == NUT_BF16 ? from_bf16(*reinterpret_cast<const uint16_t *>(p))
                                           : from_f16(*reinterpret_cast<const uint16_t *>(p));
                }
                v[r * kRun + e] = x;
            }
        }
    }
    float most = v[0];
#pragma unroll
    for (int e = 1; e < EACH; e++)
        most = fmaxf(most, v[e]);
    const float top = wave_max(most), base = top == -INFINITY ? 0.0f : top;
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < EACH; e += 4) { // four in 32 bits, whose error is an exponential's
        float four[4];
#pragma unroll
        for (int k = 0; k < 4; k++) // exp(-200) is 0 in 32 bits; what is no number stays that
            four[k] = exp_below(__builtin_elementwise_maximum(v[e + k] - base, -200.0f));
        sum += double((four[0] + four[1]) + (four[2] + four[3]));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        sum += __shfl_xor(sum, o);
    const size_t slot = size_t(row) * a.parts + part;
    if (lane == 0)
        a.stats[slot] = Part{top, 0, sum};

    // The keep largest. A bound first: the keep-th largest of the lanes' own largest,
    // below which none of them is; then all keys from it on, few where the largest are
    // spread over the lanes, at most keep lanes' where they are not.
    const uint32_t keep = a.to.beams;
    const auto at = [&](int e) {
        return part * kPart + (e / kRun * kWave + lane) * kRun + e % kRun;
    };
    // Logits of minus infinity, and what is behind the vocabulary, are no candidates.
    const auto key = [&](int e) { return v[e] > -INFINITY ? key_of(v[e], at(e)) : 0; };
    uint32_t left = most > -INFINITY ? uint32_t(key_of(most, 0) >> 32) : 0, bound = 0;
    if (keep < uint32_t(kWave)) {
        for (uint32_t k = 0; k < keep; k++) { // equal ones go together: a lower bound then
            bound = wave_most(left);
            left = left == bound ? 0 : left;
        }
    } else {
        bound = ~wave_most(~left); // the least of 64
    }
    const bool few = bound == 0; // fewer lanes than that have any
    const float least = few ? -INFINITY : logit_of(uint64_t(bound) << 32);
    __shared__ uint64_t found[kFound];
    uint32_t count = 0;
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        if (!__any(v[e] >= least && (!few || v[e] > -INFINITY)))
            continue;
        const uint64_t k = key(e);
        const bool in = k != 0 && uint32_t(k >> 32) >= bound;
        const uint64_t those = __ballot(in);
        const uint32_t to = count + __popcll(those & ((uint64_t(1) << lane) - 1));
        if (in && to < uint32_t(kFound))
            found[to] = k;
        count += uint32_t(__popcll(those));
    }
    uint64_t kept = 0; // the lane-th largest
    if (count <= uint32_t(kWave)) {
        __syncthreads();
        const uint64_t own = lane < count ? found[lane] : 0;
        uint32_t above = 0;
        for (uint32_t k = 0; k < count; k++)
            above += lane_of(own, k) > own;
        __syncthreads();
        if (lane < count)
            found[above] = own; // keys differ by their tokens
        __syncthreads();
        kept = lane < count ? found[lane] : 0;
    } else { // one after another: each lane's largest left, and the wave's
        uint64_t now = ~uint64_t(0), mine = now;
        for (uint32_t k = 0; k < keep; k++) {
            if (mine == now) {
                mine = 0;
#pragma unroll
                for (int e = 0; e < EACH; e++) {
                    const uint64_t x = key(e);
                    if (x < now && x > mine)
                        mine = x;
                }
            }
            now = wave_most(mine);
            if (now == 0)
                break;
            if (lane == k)
                kept = now;
        }
    }
    if (lane < keep)
        a.best[slot * keep + lane] = kept;
}

// A request's beams and candidates. exp and power in 64 bits: a few for each request.
//
// A part's first key is its best, so that the keep-th best of 64 groups of firsts is
// a rank that no candidate of the answer is below: the keys from it on are few where
// logits spread, and each counts those before it. Where there are more (equal
// logits), a beam's parts are merged first, one key after another, and then the
// beams. Latency bounds both: 2 requests of 10 beams, 26,160 logits, 18 best 10 us where
// merging alone took 32; 64 requests of 8 beams, 100,003 logits, 8 best 10.6 (8.6 at
// least) for 17.
struct Found {
    uint64_t rank, key;
    uint32_t beam;
};

__global__ __launch_bounds__(1024) void choose_kernel(BeamArgs a, uint32_t room)
{
    extern __shared__ uint64_t lists[]; // kMostListed words: places of parts, or a wave's lists
    __shared__ union {
        uint64_t first[kMostBeams * kMostParts]; // ranks of the parts' first keys
        uint64_t best[kMostBeams][kMostBeams];
    } lds;
    __shared__ Found found[kChosen];
    __shared__ uint32_t parts_in, count;
    __shared__ double score_of[kMostBeams], top_of[kMostBeams], log_of[kMostBeams];
    __shared__ double divisor[kMostBeams];
    __shared__ int grown[kMostBeams], state[kMostBeams]; // state: 0 none, 1 lives, 2 has ended
    const uint32_t request = blockIdx.x, beams = a.from.beams, keep = a.to.beams;
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const uint32_t waves = blockDim.x / kWave, firsts = beams * a.parts;
    // the difference to the largest logit first: it is small, or says that nothing is
    const auto scored = [&](uint32_t i, uint64_t key) {
        return score_of[i] + (double(logit_of(key)) - top_of[i] - log_of[i]);
    };
    const auto rank_of = [&](uint32_t i, uint64_t key) {
        return key == 0 ? uint64_t(0) : rank_key(scored(i, key) / divisor[i]);
    };
    // An ended beam's only candidate.
    const uint64_t over = key_of(0.0f, uint32_t(a.eos));
    if (threadIdx.x == 0)
        parts_in = count = 0;
    for (uint32_t i = wave; i < beams; i += waves) {
        const size_t row = size_t(request) * beams + i;
        const float score = a.from.scores[row];
        const bool ended = a.from.ended != nullptr && a.from.ended[row] != 0;
        const int length = a.from.lengths == nullptr ? 0 : a.from.lengths[row];
        const bool live = score > -INFINITY && !ended, mine = live && lane < a.parts;
        Part part{-INFINITY, 0, 0.0};
        uint64_t key = lane == 0 && ended ? over : 0;
        if (mine) {
            part = a.stats[row * a.parts + lane];
            key = a.best[(row * a.parts + lane) * keep];
        }
        const float top = live ? wave_max(part.most) : 0.0f;
        double sum = part.most == -INFINITY ? part.sum
                                            : part.sum * exp(double(part.most) - double(top));
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
            sum += __shfl_xor(sum, o);
        if (lane == 0) {
            grown[i] = ended ? length : length + 1;
            divisor[i] = a.power == 0.0f ? 1.0 : pow(double(max(grown[i], 1)), double(a.power));
            score_of[i] = double(score), top_of[i] = double(top);
            log_of[i] = live ? log(sum) : 0.0;
            state[i] = !(score > -INFINITY) ? 0 : ended ? 2 : 1;
        }
        wave_fence();
        if (lane < a.parts)
            lds.first[i * a.parts + lane] = score > -INFINITY ? rank_of(i, key) : 0;
    }
    __syncthreads();
    // The keep-th largest of 64 groups' largest.
    uint64_t mine = 0;
    for (uint32_t f = lane; f < firsts; f += kWave)
        mine = max(mine, lds.first[f]);
    uint32_t above = 0;
#pragma unroll
    for (int k = 0; k < kWave; k++)
        above += lane_of(mine, k) > mine;
    const bool enough = uint32_t(__popcll(__ballot(mine != 0))) >= keep;
    const uint64_t bound = enough ? ~wave_most(above < keep ? ~mine : uint64_t(0)) : 1;
    uint16_t *const places = reinterpret_cast<uint16_t *>(lists);
    for (uint32_t f = threadIdx.x; f < firsts; f += blockDim.x)
        if (lds.first[f] >= bound)
            places[atomicAdd(&parts_in, 1u)] = uint16_t(f);
    __syncthreads();
    for (uint32_t w = threadIdx.x; w < parts_in * keep; w += blockDim.x) {
        const uint32_t f = places[w / keep], k = w % keep, i = f / a.parts;
        const size_t row = size_t(request) * beams + i;
        const uint64_t key = state[i] == 1 ? a.best[(row * a.parts + f % a.parts) * keep + k]
                             : k == 0      ? over
                                           : 0;
        const uint64_t rank = rank_of(i, key);
        if (rank >= bound) {
            const uint32_t to = atomicAdd(&count, 1u);
            if (to < uint32_t(kChosen))
                found[to] = Found{rank, key, i};
        }
    }
    __syncthreads();
    const auto write = [&](uint32_t k, bool live, uint32_t beam, uint64_t key) {
        const size_t to = size_t(request) * keep + k;
        a.parents[to] = live ? int(request * beams + beam) : -1;
        a.tokens[to] = live ? int(token_of(key)) : -1;
        a.to.scores[to] = live ? float(scored(beam, key)) : -INFINITY;
        if (a.to.lengths != nullptr)
            a.to.lengths[to] = live ? grown[beam] : 0;
        if (a.to.ended != nullptr)
            a.to.ended[to] = live && (state[beam] == 2 || int(token_of(key)) == a.eos) ? 1 : 0;
    };
    if (count <= uint32_t(kChosen)) {
        if (threadIdx.x < count) {
            const Found own = found[threadIdx.x];
            uint32_t before = 0;
            for (uint32_t k = 0; k < count; k++) {
                const Found x = found[k];
                before += x.rank > own.rank ||
                          (x.rank == own.rank &&
                           (x.beam < own.beam || (x.beam == own.beam && x.key > own.key)));
            }
            if (before < keep)
                write(before, true, own.beam, own.key);
        } else if (threadIdx.x < keep) {
            write(threadIdx.x, false, 0, 0);
        }
        return;
    }
    const uint32_t merging = min(waves, kMostListed / room);
    uint64_t *list = lists + size_t(wave) * room;
    for (uint32_t i = wave; i < beams && wave < merging; i += merging) {
        const size_t row = size_t(request) * beams + i;
        uint64_t kept = lane == 0 && state[i] == 2 ? over : 0;
        if (state[i] == 1) {
            for (uint32_t k = lane; k < a.parts * keep; k += kWave)
                list[k] = a.best[row * a.parts * keep + k];
            wave_fence();
            // the heads of the parts' lists, a lane a part
            uint32_t at = 0;
            uint64_t head = lane < a.parts ? list[lane * keep] : 0;
            for (uint32_t k = 0; k < keep; k++) {
                const uint64_t now = wave_most(head);
                if (now == 0)
                    break;
                if (lane == k)
                    kept = now;
                if (head == now)
                    head = ++at < keep ? list[lane * keep + at] : 0;
            }
            wave_fence();
        }
        if (lane < keep)
            lds.best[i][lane] = kept;
    }
    __syncthreads();
    if (wave != 0)
        return;
    // the beams' lists, a lane a beam
    const auto rank = [&](uint32_t at) {
        return lane < beams && at < keep ? rank_of(lane, lds.best[lane][at]) : uint64_t(0);
    };
    uint32_t at = 0;
    uint64_t head = rank(0);
    for (uint32_t k = 0; k < keep; k++) {
        const uint64_t now = wave_most(head);
        const uint32_t beam = uint32_t(__builtin_ctzll(__ballot(head == now)));
        if (lane == beam) {
            write(k, now != 0, beam, now != 0 ? lds.best[beam][at] : 0);
            head = now != 0 ? rank(++at) : 0;
        }
    }
}

// A workgroup for 1,024 words of a row: 512 rows of 4,000 bytes 4.2 us, a launch.
template <typename Word>
__global__ __launch_bounds__(256) void gather_kernel(const char *source, size_t from_stride,
                                                     uint32_t sources, char *to, size_t to_stride,
                                                     size_t words, const int *__restrict__ parents,
                                                     int *status, uint32_t blocks)
{
    const uint32_t i = blockIdx.x / blocks, block = blockIdx.x % blocks;
    const int parent = parents[i];
    if (parent == -1)
        return;
    if (parent < 0 || uint32_t(parent) >= sources) {
        if (threadIdx.x == 0 && block == 0)
            status_flag(status, kBadParent);
        return;
    }
    const Word *x = reinterpret_cast<const Word *>(source + size_t(parent) * from_stride);
    Word *y = reinterpret_cast<Word *>(to + size_t(i) * to_stride);
    for (size_t w = size_t(block) * 256 + threadIdx.x; w < words; w += size_t(blocks) * 256)
        y[w] = x[w];
}

uint32_t parts_of(uint32_t vocab, uint32_t each)
{
    return (vocab + each * kWave - 1) / (each * kWave);
}

// Logits a lane holds, 16 to 128: the fewest whose parts fit a wave, and their
// lists its shared memory; 128 do for kMostVocab. 32 rather than 16 where that leaves
// 8,192 waves: each finds its own largest, and lists them for the second launch. Calls of
// 16, 32, 64 and 128, us, fp16: 4 beams of 32,000 logits 14.4, 15.4, 18.6, 23.6, 128 of
// them 17.2, 18.1, 20.7, 26.7, 512 of them 30.9, 29.9, 33.2, 47.1; 512 of 100,003 (32 at
// least) 57, 72, 146.
uint32_t each_of(uint32_t rows, uint32_t vocab, uint32_t keep)
{
    uint32_t each = 16;
    while (each < 128 && (parts_of(vocab, each) > kMostParts ||
                          parts_of(vocab, each) * keep > kMostListed ||
                          (each < 32 && uint64_t(rows) * parts_of(vocab, each) > 8192)))
        each *= 2;
    return each;
}

size_t carve(BeamArgs &a, char *base)
{
    const auto aligned = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
    a.parts = parts_of(a.vocab, each_of(a.from.requests * a.from.beams, a.vocab, a.to.beams));
    const size_t parts = size_t(a.from.requests) * a.from.beams * a.parts;
    a.stats = reinterpret_cast<Part *>(base);
    a.best = reinterpret_cast<uint64_t *>(base + aligned(parts * sizeof(Part)));
    return aligned(parts * sizeof(Part)) + aligned(parts * a.to.beams * sizeof(uint64_t));
}

template <int TYPE> void scan_as(const BeamArgs &a, dim3 grid, hipStream_t stream)
{
    const uint32_t each = each_of(a.from.requests * a.from.beams, a.vocab, a.to.beams);
    const auto run = each == 16   ? scan_kernel<TYPE, 16>
                     : each == 32 ? scan_kernel<TYPE, 32>
                     : each == 64 ? scan_kernel<TYPE, 64>
                                  : scan_kernel<TYPE, 128>;
    hipLaunchKernelGGL(run, grid, dim3(kWave), 0, stream, a);
}

} // namespace

size_t beam_workspace(const BeamsView &from, const BeamsView &to, uint32_t vocab)
{
    BeamArgs a{};
    a.from = from, a.to = to, a.vocab = vocab;
    const size_t bytes = carve(a, nullptr);
    paged_grid(uint64_t(from.requests) * from.beams * a.parts, kWave);
    paged_grid(from.requests, 1024);
    return bytes;
}

void launch_beam_select(const BeamsView &from, const BeamsView &to, const void *logits, int type,
                        size_t row_stride, uint32_t vocab, int eos, float power, int *parents,
                        int *tokens, char *workspace, hipStream_t stream)
{
    BeamArgs a{};
    a.from = from, a.to = to, a.logits = logits, a.row_stride = row_stride, a.vocab = vocab;
    a.eos = eos, a.power = power, a.parents = parents, a.tokens = tokens;
    carve(a, workspace);
    const uint32_t rows = from.requests * from.beams, y = std::min(rows, 32768u);
    const dim3 grid(a.parts, y, (rows + y - 1) / y);
    if (type == NUT_F32)
        scan_as<NUT_F32>(a, grid, stream);
    else if (type == NUT_F16)
        scan_as<NUT_F16>(a, grid, stream);
    else
        scan_as<NUT_BF16>(a, grid, stream);
    check_launch("beam select");
    const uint32_t room = a.parts * to.beams;
    // a wave a beam, and threads for kChosen candidates
    const uint32_t waves = std::min(std::max(from.beams, uint32_t(kChosen / kWave)), 16u);
    hipLaunchKernelGGL(choose_kernel, dim3(from.requests), dim3(waves * kWave),
                       kMostListed * sizeof(uint64_t), stream, a, room);
    check_launch("beam select");
}

void launch_beam_gather(const char *source, size_t from_stride, uint32_t sources, char *to,
                        size_t to_stride, uint32_t rows, size_t row_bytes, const int *parents,
                        int *status, hipStream_t stream)
{
    const uintptr_t all = reinterpret_cast<uintptr_t>(source) | reinterpret_cast<uintptr_t>(to) |
                          from_stride | to_stride | row_bytes;
    const bool wide = all % 16 == 0;
    const size_t words = row_bytes / (wide ? 16 : 4);
    // 4 words a thread, as far as one launch covers them
    const uint64_t most = 0xffffffffull / 256 / rows;
    const uint32_t blocks = uint32_t(std::min<uint64_t>((words + 1023) / 1024, most));
    hipLaunchKernelGGL(wide ? gather_kernel<uint4> : gather_kernel<uint32_t>, dim3(rows * blocks),
                       dim3(256), 0, stream, source, from_stride, sources, to, to_stride, words,
                       parents, status, blocks);
    check_launch("beam gather");
}

} // namespace nut
