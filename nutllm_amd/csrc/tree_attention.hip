// tree_attention.hip — attention of a tree of drafted tokens over a paged KV
// cache.
//
// The query rows of a KV head are its sequence's nodes times the heads that
// share it, node after node. Rows that the sequence held before are seen by every
// node; of a tile that reaches into the drafted rows each lane takes its node's mask.
// Few query rows, or little work: tree_kernel, whose workgroups take 16 or 32 of
// them and a run of the sequence's rows, in registers as in paged_attention.hip.
// Many: staged_kernel, whose workgroups take 64 and share rows in shared memory.
// A second launch joins the parts of either.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "paged_attend.hpp"
#include "runtime.hpp"
#include "serving.hpp"

namespace nut {

namespace {

constexpr uint32_t kPieceRows = 1024; // rows whose offsets are in shared memory at once

struct TreeArgs {
    PagedView kv;
    PagedSeqs s;
    DraftView d;
    const float *query;
    size_t query_stride;
    uint32_t heads, group;
    float scale; // times log2(e)
    float *out, *lse;
    uint32_t blocks, run, runs, units; // of tree_kernel
    uint32_t shares;                   // of staged_kernel
    uint32_t teams;                    // of a query row, of the joins
    bool past;                         // rows go past the caches' replacement
    uint64_t *before; // [batch + 1]: stages before each sequence
    // tree_kernel: [total][heads][runs], of every query row and run; staged_kernel:
    // [2 shares][kBlock], of the query rows of the items that a share cuts
    float *parts;  // [head_dim] each, unnormalised
    float2 *stats; // exponent they refer to, sum
};

// Rows of the sequence and of its nodes together; 0, reported once, where the
// length is not one that the call allows.
__device__ __forceinline__ uint32_t rows_of(const TreeArgs &a, uint32_t b, uint32_t nodes,
                                            uint32_t &held, bool report)
{
    const int n = a.s.lengths[b];
    held = 0;
    if (!length_with(n, nodes, a.s.max_length)) {
        if (report)
            status_flag(a.kv.status, kBadLength);
        return 0;
    }
    held = uint32_t(n);
    return held + nodes;
}

// Not finite: a 16-bit pair, or an fp32 value.
template <int TYPE> __device__ __forceinline__ bool odd_word(uint32_t w)
{
    if constexpr (TYPE == NUT_F32)
        return (w & 0x7f800000u) == 0x7f800000u;
    const uint32_t e = TYPE == NUT_F16 ? 0x7c00u : 0x7f80u;
    return (w & e) == e || (w >> 16 & e) == e;
}

// One component of a row.
template <int TYPE> __device__ __forceinline__ float component(const char *row, uint32_t d)
{
    if constexpr (TYPE == NUT_F32)
        return reinterpret_cast<const float *>(row)[d];
    const uint32_t bits = reinterpret_cast<const uint16_t *>(row)[d];
    return TYPE == NUT_BF16 ? from_bf16(bits) : from_f16(bits);
}

// A tile against 16 query rows. `gone`: rows that no node sees, the same in every
// lane; `seen`: with `drafted`, the rows that the lane's node sees.
template <int TYPE, int HD, bool FULL>
__device__ __forceinline__ void attend_tree(Tile<TYPE, HD> &tile, const size_t *at, uint32_t gone,
                                            bool drafted, uint32_t seen,
                                            const Query<TYPE, HD> &q, Softmax<TYPE, HD> &sm,
                                            const PagedView &kv, int lane)
{
    using T = Tile<TYPE, HD>;
    constexpr int G = T::G, E = T::kEach;
    const int j = lane >> 4;
    float s[T::kScores];
    score<TYPE, HD>(tile, q, s);
    uint32_t odd = 0; // rows with values that are not finite, which not every node may see
    if (gone != 0 || drafted) {
        const uint32_t none = gone >> (4 * j);
#pragma unroll
        for (int r = 0; r < T::kScores; r++) {
            const int bit = 16 * (r / 4) + r % 4;
            const bool out = none >> bit & 1;
            bool strange = false;
#pragma unroll
            for (int w = 0; w < T::kWords; w++) {
                tile.v[r][w] = out ? 0 : tile.v[r][w];
                strange = strange || odd_word<TYPE>(tile.v[r][w]);
            }
            s[r] = out || !(seen >> (4 * j) >> bit & 1) ? -INFINITY : s[r];
            if (drafted) {
                const uint64_t any = __ballot(strange);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    odd |= (any >> (16 * i) & 0xffff) != 0 ? 1u << (bit + 4 * i) : 0;
            }
        }
        odd = __builtin_amdgcn_readfirstlane(odd);
    }
    float p[8];
    float most = s[0];
#pragma unroll
    for (int r = 1; r < T::kScores; r++)
        most = fmaxf(most, s[r]);
    sm.raise(max_over_rows(most));
#pragma unroll
    for (int r = 0; r < T::kScores; r++) {
        p[r] = __builtin_amdgcn_exp2f(s[r] - sm.ref);
        sm.sum += p[r];
    }
    if (odd != 0) {
        // 0 times what is not finite is no number: such rows leave the product,
        // and nodes that weigh them add them one by one.
        for (uint32_t left = odd; left != 0; left &= left - 1) {
            const int row = __builtin_ctz(left), own = row % 16 / 4;
            const char *v = kv.values + at[row];
            float weight = 0.0f;
#pragma unroll
            for (int r = 0; r < T::kScores; r++)
                if (16 * (r / 4) + r % 4 == row - 4 * own)
                    weight = p[r];
            weight = __shfl(weight, 16 * own + (lane & 15));
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t d = 16 * (g / E * E) + 4 * j * E + i * E + g % E;
                    if (weight != 0.0f && (FULL || d < kv.head_dim))
                        sm.o[g][i] = fmaf(weight, component<TYPE>(v, d), sm.o[g][i]);
                }
        }
#pragma unroll
        for (int r = 0; r < T::kScores; r++)
#pragma unroll
            for (int w = 0; w < T::kWords; w++)
                tile.v[r][w] = odd >> (16 * (r / 4) + r % 4 + 4 * j) & 1 ? 0 : tile.v[r][w];
    }
    if constexpr (T::kWide) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int g = 0; g < G; g++)
                sm.o[g] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                    __uint_as_float(tile.v[r][g]), p[r], sm.o[g], 0, 0, 0);
    } else {
        constexpr int kLimbs = Query<TYPE, HD>::kLimbs;
        u32x4 limb[kLimbs];
        split<TYPE, kLimbs>(p, limb);
#pragma unroll
        for (int g = 0; g < G; g++) {
            const u32x4 x = tile.component(g);
#pragma unroll
            for (int l = kLimbs - 1; l >= 0; l--)
                sm.o[g] = product<TYPE>(x, limb[l], sm.o[g]);
        }
    }
}

// WQ of a workgroup's waves hold different query rows, and share their rows' offsets;
// the others take tiles of rows in turn. Latency bounds it: 16 nodes of 32 heads of 64
// over 211 fp32 rows take 7.4 us (6.0 at least), two tiles a wave one after another.
template <int HD> constexpr int kTreeWaves = HD == 256 ? 2 : 4;

template <int TYPE, int HD, bool FULL, int WQ>
__global__ __launch_bounds__(64 * kTreeWaves<HD>, HD == 256 ? 1 : 2) void tree_kernel(TreeArgs a)
{
    using T = Tile<TYPE, HD>;
    constexpr int G = T::G, WAVES = kTreeWaves<HD>, kThreads = 64 * WAVES;
    constexpr int WK = WAVES / WQ;
    constexpr int kStride = HD + 4;
    __shared__ union Shared {
        size_t at[kPieceRows];
        float o[WAVES][16][kStride];
    } lds;
    __shared__ float stat[3][WAVES][16];
    __shared__ uint32_t gone[kPieceRows / 32];
    const PagedView &kv = a.kv;
    // Workgroups go to the 8 XCDs in turn: the blocks that read the same rows
    // follow one another on one of them.
    const uint32_t turn = blockIdx.x / 8;
    const uint32_t unit = turn / a.blocks * 8 + blockIdx.x % 8, block = turn % a.blocks;
    if (unit >= a.units)
        return;
    const uint32_t c = unit % a.runs, h = unit / a.runs % kv.kv_heads;
    const uint32_t b = unit / a.runs / kv.kv_heads;
    const bool leader = threadIdx.x == 0 && c == 0 && h == 0 && block == 0;
    const NodeSpan nodes = nodes_of(a.d, b, leader);
    const uint32_t queries = nodes.count * a.group, begins = block * 16 * WQ;
    if (begins >= queries)
        return;
    uint32_t held;
    const uint32_t total = rows_of(a, b, nodes.count, held, leader);
    const uint32_t begin = c * a.run;
    if (begin >= total && (c != 0 || a.parts != nullptr))
        return;
    const uint32_t count = min(total - begin, a.run);

    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int j = lane >> 4, column = lane & 15;
    const int wq = wave % WQ, wk = wave / WQ;
    const uint32_t first = begins + wq * 16; // of the wave's query rows
    const bool valid = first + column < queries;
    const uint32_t query = valid ? first + column : begins;
    const uint32_t node = nodes.from + query / a.group, head = h * a.group + query % a.group;
    Query<TYPE, HD> q;
    q.fetch(a.query + node * a.query_stride + size_t(head) * kv.head_dim, valid, kv.head_dim,
            lane);
    const uint32_t *mask = a.d.mask + node * a.d.mask_stride;
    const uint32_t words = (nodes.count + 31) / 32;
    q.convert(a.scale);

    Softmax<TYPE, HD> sm;
    for (uint32_t piece = 0; piece < count; piece += kPieceRows) {
        const uint32_t rows = min(count - piece, kPieceRows);
        if (piece != 0)
            __syncthreads();
        for (uint32_t i = threadIdx.x; i < (rows + 63) / 64 * 64; i += kThreads) {
            const uint32_t row = begin + piece + i;
            size_t at = 0;
            bool out = i >= rows;
            if (!out) {
                const uint32_t index = page_of(kv, row);
                at = paged_row(kv, a.s, b, index, row - index * kv.page_size, h);
                out = at == kNoRow;
            }
            lds.at[i] = out ? 0 : at;
            const uint64_t masked = __ballot(out);
            if (lane % 32 == 0)
                gone[i / 32] = uint32_t(masked >> lane);
        }
        __syncthreads();
        constexpr uint32_t kAll = T::kWide ? 0xffffu : 0xffffffffu;
        const int tiles = first >= queries ? 0 : int((rows + T::kRows - 1) / T::kRows);
        for (int t = wk; t < tiles; t += WK) {
            Tile<TYPE, HD> x;
            x.template load<FULL, false>(kv, lds.at + t * T::kRows, lane);
            const uint32_t none = uint32_t(__builtin_amdgcn_readfirstlane(
                gone[t * T::kRows / 32] >> (t * T::kRows % 32) & kAll));
            const uint32_t row = begin + piece + t * T::kRows;
            const bool drafted = row + T::kRows > held;
            const uint32_t seen = !drafted ? ~0u
                                           : mask_bits(int64_t(row) - held, words,
                                                       [&](uint32_t w) { return mask[w]; });
            attend_tree<TYPE, HD, FULL>(x, lds.at + t * T::kRows, none, drafted, seen, q, sm, kv,
                                        lane);
        }
    }

    // The waves' sums side by side; then a thread per four components adds those of
    // the same query rows.
    const uint32_t parts = FULL ? HD / 4 : kv.head_dim / 4;
    sm.sum += __shfl_xor(sm.sum, 16);
    sm.sum += __shfl_xor(sm.sum, 32);
    __syncthreads();
    if (j == 0)
        stat[0][wave][column] = sm.most, stat[1][wave][column] = sm.ref,
        stat[2][wave][column] = sm.sum;
    constexpr int E = T::kEach;
#pragma unroll
    for (int p = 0; p < G; p += E) {
        float flat[4 * E]; // components 16 p + 4 j E .. of the lane's query row
#pragma unroll
        for (int g = 0; g < E; g++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                flat[i * E + g] = sm.o[p + g][i];
        float *to = lds.o[wave][column] + 16 * p + 4 * j * E;
#pragma unroll
        for (int d = 0; d < 4 * E; d += 4)
            *reinterpret_cast<f32x4 *>(to + d) =
                f32x4{flat[d], flat[d + 1], flat[d + 2], flat[d + 3]};
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < WQ * 16 * parts; i += kThreads) {
        const uint32_t k = i / parts, d = (i - k * parts) * 4, of = k / 16, c16 = k % 16;
        const uint32_t row = begins + of * 16 + c16;
        if (row >= queries)
            continue;
        float most = stat[0][of][c16];
#pragma unroll
        for (int w = 1; w < WK; w++)
            most = fmaxf(most, stat[0][of + w * WQ][c16]);
        const float ref = most == -INFINITY ? 0.0f : most - Softmax<TYPE, HD>::kShift;
        float sum = 0.0f;
        f32x4 o{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < WK; w++) {
            const int from = of + w * WQ;
            // what no row of a finite score reached is zero, or not a number
            const float f = stat[0][from][c16] == -INFINITY
                                ? 1.0f
                                : __builtin_amdgcn_exp2f(stat[1][from][c16] - ref);
            sum = fmaf(stat[2][from][c16], f, sum);
            const f32x4 y = *reinterpret_cast<const f32x4 *>(&lds.o[from][c16][d]);
#pragma unroll
            for (int e = 0; e < 4; e++)
                o[e] = fmaf(y[e], f, o[e]);
        }
        const size_t at = size_t(nodes.from + row / a.group) * a.heads + h * a.group +
                          row % a.group;
        if (a.parts != nullptr) {
            *reinterpret_cast<f32x4 *>(a.parts + (at * a.runs + c) * kv.head_dim + d) = o;
            if (d == 0)
                a.stats[at * a.runs + c] = make_float2(sum == 0.0f ? -INFINITY : ref, sum);
        } else {
            *reinterpret_cast<f32x4 *>(a.out + at * kv.head_dim + d) =
                sum == 0.0f ? f32x4{0, 0, 0, 0} : o * (1.0f / sum);
            if (d == 0 && a.lse != nullptr)
                a.lse[at] = sum == 0.0f ? -INFINITY : (ref + log2f(sum)) * 0.69314718055994531f;
        }
    }
}

// ---------------------------------------------------------------- staged --

// Many query rows: the four waves hold 16 each and share every tile of rows, staged
// in shared memory. 16-bit rows come by DMA, the next stage while this one
// is multiplied; fp32 rows come through registers and are kept as three bfloat16
// limbs, whose six largest products with the query's limbs leave out 2^-21 of a
// product at most and 2^-24 in the mean: 2.7 times the rate of the fp32
// instruction. Keys are read as they lie; values by the transposing read, of the
// keys that the lane's weights are of, so that those need no exchange.
template <int TYPE, int HD> struct Stage {
    static constexpr int kPlanes = TYPE == NUT_F32 ? 3 : 1;
    static constexpr int kType = TYPE == NUT_F32 ? NUT_BF16 : TYPE; // of the planes
    static constexpr int kRows = HD <= 64 && TYPE != NUT_F32 ? 64 : 32;
    static constexpr int kChunks = HD <= 32 ? 4 : HD <= 64 ? 8 : HD <= 128 ? 16 : 32; // of a row
    static constexpr int kUsed = HD / 8;
    // The stage at work and, of 16-bit rows, the one that is fetched beside it. (Two
    // fetched ahead, at a row of 128 components, read no faster: 418 us for 408 of
    // four sequences of up to 32,768 fp16 rows, 32 KV heads.)
    static constexpr int kBuffers = TYPE == NUT_F32 ? 1 : 2;
    static constexpr int kBytes = kPlanes * kRows * kChunks * 16; // of keys, or of values
    // Chunks of 16 bytes trade places within 128, by the row: 16 rows of one chunk
    // lie on all banks.
    static constexpr int kShift = kChunks < 8 ? 3 : kChunks == 8 ? 3 : kChunks == 16 ? 4 : 5;
    static __device__ __forceinline__ uint32_t place(uint32_t i) { return i ^ (i >> kShift & 7); }
    static __device__ __forceinline__ uint32_t offset(uint32_t row, uint32_t chunk)
    {
        return place(row * kChunks + chunk) * 16;
    }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// BYTES (16 or 4) for each lane, from `source` to shared memory, lane after lane.
// As asm: the compiler would wait for all of it before it reads shared memory.
template <int BYTES = 16, bool NT = false>
__device__ __forceinline__ void stage_dma(const void *source, const void *to)
{
    const uint32_t at = __builtin_amdgcn_readfirstlane(uint32_t(
        reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void *)to)));
    if constexpr (BYTES == 16 && NT)
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt"
                     :
                     : "v"(source), "s"(at)
                     : "memory", "m0");
    else if constexpr (BYTES == 16)
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                     :
                     : "v"(source), "s"(at)
                     : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
                     :
                     : "v"(source), "s"(at)
                     : "memory", "m0");
}

// Whether a component of an fp32 row is no number, whatever its bits.
__device__ __forceinline__ bool no_number(const char *row, uint32_t head_dim)
{
    bool found = false;
#pragma unroll 1
    for (uint32_t d = 0; d < head_dim; d += 8) {
        float x[8];
        load8<NUT_F32>(row + d * 4, x);
#pragma unroll
        for (int e = 0; e < 8; e++)
            found = found || x[e] != x[e];
    }
    return found;
}

// A compiler that has the loads before this does not put them off behind it.
__device__ __forceinline__ void keep_loads() { asm volatile("" ::: "memory"); }

// A stage against 16 query rows; the other arguments as attend_tree's, a word for
// 32 rows. `odd`: rows some of whose values are not finite and were
// staged as 0; they are added one by one. Shared memory answers after 100 cycles
// and a product after 30, so that everything that can be is asked for together:
// all keys of a plane, the values before the softmax, and products in turn that do
// not wait for one another.
template <int TYPE, int HD, bool FULL>
__device__ __forceinline__ void
attend_stage(const char *keys, const char *values, const size_t *at,
             const uint32_t (&gone)[Stage<TYPE, HD>::kRows / 32], bool drafted,
             const uint32_t (&odd)[Stage<TYPE, HD>::kRows / 32],
             const uint32_t (&seen)[Stage<TYPE, HD>::kRows / 32],
             const Query<Stage<TYPE, HD>::kType, HD> &q,
             Softmax<Stage<TYPE, HD>::kType, HD> &sm, const PagedView &kv, int lane)
{
    using S = Stage<TYPE, HD>;
    constexpr int G = HD / 16, kParts = HD / 32, kType = S::kType, kPlanes = S::kPlanes;
    constexpr int kLimbs = Query<kType, HD>::kLimbs, kSubs = S::kRows / 16, kHalves = kSubs / 2;
    const uint32_t j = lane >> 4, c = lane & 15;
    const auto key = [&](int p, int sub, int n) {
        return *reinterpret_cast<const u32x4 *>(
            keys + S::offset(p * S::kRows + sub * 16 + c, n * 4 + j));
    };
    f32x4 acc[kSubs];
#pragma unroll
    for (int sub = 0; sub < kSubs; sub++)
        acc[sub] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int p = kPlanes - 1; p >= 0; p--) {
        u32x4 k[kSubs][kParts];
#pragma unroll
        for (int n = 0; n < kParts; n++)
#pragma unroll
            for (int sub = 0; sub < kSubs; sub++)
                k[sub][n] = key(p, sub, n);
        keep_loads();
#pragma unroll
        for (int n = 0; n < kParts; n++)
#pragma unroll
            for (int l = kLimbs - 1; l >= 0; l--)
#pragma unroll
                for (int sub = 0; sub < kSubs; sub++)
                    if (kPlanes == 1 || p + l < 3)
                        acc[sub] = product<kType>(k[sub][n], q.x[n][l], acc[sub]);
    }
    // Values of plane p, kGroup tiles of 16 components from tile g0 on: of rows
    // 4 j + c / 4 (then 16 further), components 16 g + 4 (c % 4) onwards, transposed.
    constexpr int kGroup = kHalves * G <= 8 ? G : G / 2;
    u32x4 v[kHalves][kGroup];
    const auto load_values = [&](int p, int g0) {
#pragma unroll
        for (int g = 0; g < kGroup; g++)
#pragma unroll
            for (int half = 0; half < kHalves; half++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t row = p * S::kRows + half * 32 + 16 * e + 4 * j + c / 4;
                    const char *from =
                        values + S::offset(row, 2 * (g0 + g) + (c & 3) / 2) + (c & 1) * 8;
                    const u32x2 z = __builtin_bit_cast(
                        u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)from));
                    v[half][g][2 * e] = z[0], v[half][g][2 * e + 1] = z[1];
                }
        keep_loads();
    };
    load_values(kPlanes - 1, 0);
    float s[kHalves][8];
    float all = 0.0f; // not a number after one that is none
#pragma unroll
    for (int sub = 0; sub < kSubs; sub++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            all += acc[sub][i];
    if (__any(all != all)) {
        // An infinite key: the first limbs' product has the sum's sign, later ones
        // of zero, or of the other sign, make it no number. (So do sums of both
        // infinities, which are none in the end either.) A NaN may look infinite in
        // its upper limb: fp32 keys are read again, a lane a row.
        uint32_t none = 0; // rows of the lane whose keys are no numbers
        if constexpr (TYPE == NUT_F32) {
            static_assert(S::kRows == 32, "a bit a row");
            const size_t row = at[lane % 32];
            const bool is = row != kNoRow && no_number(kv.keys + row, kv.head_dim);
            none = uint32_t(__ballot(is)) >> (4 * j);
        }
#pragma unroll
        for (int sub = 0; sub < kSubs; sub++) {
            f32x4 first{0, 0, 0, 0};
#pragma unroll
            for (int n = 0; n < kParts; n++)
                first = product<kType>(key(0, sub, n), q.x[n][0], first);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float x = none >> (16 * sub + i) & 1 ? __builtin_nanf("") : first[i];
                acc[sub][i] = acc[sub][i] != acc[sub][i] ? x : acc[sub][i];
            }
        }
    }
#pragma unroll
    for (int half = 0; half < kHalves; half++)
#pragma unroll
        for (int r = 0; r < 8; r++) {
            const float x = acc[2 * half + r / 4][r % 4];
            s[half][r] = kType == NUT_F16 ? ldexpf(x, q.exponent) : x;
        }
    bool masked = drafted;
#pragma unroll
    for (int half = 0; half < kHalves; half++)
        masked = masked || gone[half] != 0;
    if (masked)
#pragma unroll
        for (int half = 0; half < kHalves; half++) {
            const uint32_t mine = (seen[half] & ~gone[half]) >> (4 * j);
#pragma unroll
            for (int r = 0; r < 8; r++)
                s[half][r] = mine >> (16 * (r / 4) + r % 4) & 1 ? s[half][r] : -INFINITY;
        }
    u32x4 limb[kHalves][kLimbs];
    float p[kHalves][8];
    float most = s[0][0];
#pragma unroll
    for (int half = 0; half < kHalves; half++)
#pragma unroll
        for (int r = 0; r < 8; r++)
            most = fmaxf(most, s[half][r]);
    sm.raise(max_over_rows(most));
    float sum[kHalves][2] = {};
#pragma unroll
    for (int half = 0; half < kHalves; half++) {
#pragma unroll
        for (int r = 0; r < 8; r++) {
            p[half][r] = __builtin_amdgcn_exp2f(s[half][r] - sm.ref);
            sum[half][r % 2] += p[half][r];
        }
        split<kType, kLimbs>(p[half], limb[half]);
        sm.sum += sum[half][0] + sum[half][1];
    }
#pragma unroll
    for (int half = 0; half < kHalves; half++)
        for (uint32_t left = odd[half]; left != 0; left &= left - 1) {
            const int row = __builtin_ctz(left), own = row % 16 / 4;
            const char *from = kv.values + at[half * 32 + row];
            float weight = 0.0f;
#pragma unroll
            for (int r = 0; r < 8; r++)
                if (16 * (r / 4) + r % 4 == row - 4 * own)
                    weight = p[half][r];
            weight = __shfl(weight, 16 * own + c);
            for (int g = 0; g < G; g++) // rare: not unrolled but for the sums
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t d = 16 * g + 4 * j + i;
                    const float x = FULL || d < kv.head_dim ? component<TYPE>(from, d) : 0.0f;
                    const bool adds = weight != 0.0f && !(fabsf(x) < INFINITY);
#pragma unroll
                    for (int k = 0; k < G; k++)
                        if (k == g && adds)
                            sm.o[k][i] = fmaf(weight, x, sm.o[k][i]);
                }
        }
#pragma unroll
    for (int pl = kPlanes - 1; pl >= 0; pl--)
#pragma unroll
        for (int g0 = 0; g0 < G; g0 += kGroup) {
            if (pl != kPlanes - 1 || g0 != 0)
                load_values(pl, g0);
#pragma unroll
            for (int half = 0; half < kHalves; half++)
#pragma unroll
                for (int l = kLimbs - 1; l >= 0; l--)
#pragma unroll
                    for (int g = 0; g < kGroup; g++)
                        if (kPlanes == 1 || pl + l < 3)
                            sm.o[g0 + g] =
                                product<kType>(v[half][g], limb[half][l], sm.o[g0 + g]);
        }
}

constexpr uint32_t kBlock = 64; // query rows of a workgroup
// Stages that a workgroup takes at least. One, two and four, us: 64 nodes of 32 heads of
// 64 on 4 KV heads, one sequence of 1,000 bfloat16 rows 20.5, 22.0, 24.6, of fp32 ones
// 23.7, 22.8, 24.7; 16 sequences of 100 29.6, 26.4, 28.1.
constexpr uint32_t kLeast = 2;

// How the work is shared out. An item is a block of a sequence's query rows and a
// KV head, its work the stages of the sequence's rows; items follow one another
// by sequence, KV head and block, and `shares` workgroups take equal parts of all
// stages, wherever that cuts an item: lengths and trees are known to the device
// alone, and parts by the longest would leave most of the chip without work (16
// sequences of 1 to 2,048 rows: 47 us, of which a CU worked half).
struct Item {
    NodeSpan nodes;
    uint32_t held, total, blocks, stages;
};

template <int R>
__device__ __forceinline__ Item item_of(const TreeArgs &a, uint32_t b, bool report)
{
    Item it;
    it.nodes = nodes_of(a.d, b, report);
    it.total = rows_of(a, b, it.nodes.count, it.held, report && it.nodes.count != 0);
    it.blocks = (it.nodes.count * a.group + kBlock - 1) / kBlock;
    it.stages = max((it.total + R - 1) / R, 1u); // a sequence out of range gets zeros
    return it;
}

struct Shares {
    uint64_t all; // stages
    uint32_t count;
    __device__ __forceinline__ uint64_t begin(uint32_t i) const { return all * i / count; }
    // The share that stage x, below `all`, is of.
    __device__ __forceinline__ uint32_t of(uint64_t x) const
    {
        uint32_t i = uint32_t(x * count / all);
        while (i + 1 < count && begin(i + 1) <= x)
            i++;
        while (begin(i) > x)
            i--;
        return i;
    }
};

__device__ __forceinline__ uint32_t share_count(uint64_t all, uint32_t most)
{
    return uint32_t(max(min((all + kLeast - 1) / kLeast, uint64_t(most)), uint64_t(1)));
}

// The stages before each sequence: a thread sums those of `each` sequences, and
// then the threads' sums are summed. Returns the share-out, and in `before` the
// stages before this thread's first sequence. 256 threads.
template <int R>
__device__ __forceinline__ Shares share_out(const TreeArgs &a, uint32_t each, bool report,
                                            uint64_t &before)
{
    __shared__ uint64_t sums[4];
    uint64_t mine = 0;
    for (uint32_t k = 0; k < each; k++) {
        const uint32_t b = threadIdx.x * each + k;
        if (b >= a.s.batch)
            break;
        const Item it = item_of<R>(a, b, report);
        mine += uint64_t(it.blocks) * it.stages;
    }
    mine *= a.kv.kv_heads;
    uint64_t upto = mine;
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const uint64_t x = uint64_t(__shfl_up((unsigned long long)upto, o));
        upto += lane >= uint32_t(o) ? x : 0;
    }
    if (lane == kWave - 1)
        sums[wave] = upto;
    __syncthreads();
    Shares shares{0, 1};
    before = upto - mine;
    for (uint32_t w = 0; w < 4; w++) {
        before += w < wave ? sums[w] : 0;
        shares.all += sums[w];
    }
    shares.count = share_count(shares.all, a.shares);
    return shares;
}

// Workgroups that a CU holds, by registers and shared memory.
constexpr int staged_groups(int type, uint32_t head_dim)
{
    if (head_dim <= 64)
        return 3;
    return (head_dim <= 128 ? 3 : 2) - (type == NUT_F32 ? 1 : 0);
}

// 64 nodes of 32 heads of 64 on 4 KV heads, bfloat16: 16 sequences of 1 to 2,048 rows 32
// us, a third of them the matrix instructions'; 32 of 4,096 149, 460 TFLOP/s of useful
// products, three limbs each: between the products stand the softmax and the splitting
// of its weights. 203 nodes of 24 heads of 80 on 3, fp32, 7 sequences of up to 5,001
// rows: 220, half of it the rows' splitting into limbs. 32 heads of 128, fp16, 4
// sequences of 24,000 to 32,768 rows: 400, 4.9 TB/s.
template <int TYPE, int HD, bool FULL>
__global__ __launch_bounds__(256, staged_groups(TYPE, HD)) void staged_kernel(TreeArgs a)
{
    using S = Stage<TYPE, HD>;
    constexpr int G = HD / 16, R = S::kRows;
    constexpr uint32_t kEach = 4, kPiece = kEach * R; // rows whose offsets are found at once
    constexpr int kWork = R * S::kChunks / 256; // chunks of a plane a thread
    static_assert(R * S::kChunks % 256 == 0 || R * S::kChunks < 256, "whole chunks a thread");
    __shared__ alignas(128) char stage[S::kBuffers][2][S::kBytes];
    __shared__ size_t offsets[2][kPiece];
    __shared__ int table[kPiece];
    __shared__ uint32_t gone[2][kPiece / 32], strange[2][2];
    __shared__ uint64_t where[2]; // a sequence, and the stages before it
    const PagedView &kv = a.kv;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t j = lane >> 4, column = lane & 15;
    const uint32_t used = FULL ? S::kUsed : kv.head_dim / 8;
    if constexpr (!FULL && TYPE != NUT_F32) // where no chunk of a row comes to
        for (uint32_t i = threadIdx.x; i < sizeof stage / 16; i += 256)
            reinterpret_cast<u32x4 *>(stage)[i] = u32x4{0, 0, 0, 0};

    const uint32_t each = (a.s.batch + 255) / 256;
    uint64_t before;
    const Shares shares = share_out<R>(a, each, blockIdx.x == 0, before);
    // Workgroups go to the 8 XCDs in turn: each takes shares that follow one another,
    // so that the blocks that read the same rows do so through one cache.
    const uint32_t run_of = (shares.count + 7) / 8;
    const uint32_t share = blockIdx.x % 8 * run_of + blockIdx.x / 8;
    if (blockIdx.x / 8 >= run_of || share >= shares.count ||
        (shares.all == 0 && blockIdx.x != 0))
        return;
    uint64_t at_stage = shares.begin(share);
    const uint64_t end_stage = shares.begin(share + 1);
    if (blockIdx.x == 0) { // for the join
        uint64_t upto = before;
        for (uint32_t k = 0; k < each; k++) {
            const uint32_t b = threadIdx.x * each + k;
            if (b >= a.s.batch)
                break;
            const Item it = item_of<R>(a, b, false);
            a.before[b] = upto;
            upto += uint64_t(it.blocks) * it.stages * kv.kv_heads;
        }
        if (threadIdx.x == 0)
            a.before[a.s.batch] = shares.all;
    }
    for (uint32_t k = 0; k < each; k++) { // one thread has the sequence that holds it
        const uint32_t b = threadIdx.x * each + k;
        if (b >= a.s.batch || before > at_stage)
            break;
        const Item it = item_of<R>(a, b, false);
        const uint64_t work = uint64_t(it.blocks) * it.stages * kv.kv_heads;
        if (at_stage < before + work) {
            where[0] = b, where[1] = before;
            break;
        }
        before += work;
    }
    __syncthreads();
    uint32_t b = uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(where[0])));
    uint64_t passed = where[1]; // stages before sequence b
    bool opening = true;

    while (at_stage < end_stage) {
        const Item it = item_of<R>(a, b, false);
        const uint64_t work = uint64_t(it.blocks) * it.stages * kv.kv_heads;
        if (at_stage >= passed + work) {
            passed += work;
            b++;
            continue;
        }
        const uint32_t item = uint32_t((at_stage - passed) / it.stages);
        const uint32_t from_stage = uint32_t(at_stage - passed - uint64_t(item) * it.stages);
        const uint32_t to_stage =
            uint32_t(min(uint64_t(it.stages), from_stage + (end_stage - at_stage)));
        const bool cut = from_stage != 0 || to_stage != it.stages;
        const uint32_t slot = 2 * share + (opening && from_stage != 0 ? 0 : 1);
        opening = false;
        at_stage += to_stage - from_stage;
        const uint32_t h = item / it.blocks, block = item - h * it.blocks;
        const NodeSpan nodes = it.nodes;
        const uint32_t held = it.held;
        const uint32_t queries = nodes.count * a.group, begins = block * kBlock;
        const uint32_t begin = from_stage * R, count = min(to_stage * R, it.total) - begin;
        const uint32_t first = begins + wave * 16; // of the wave's query rows
        const bool valid = first + column < queries;
        const uint32_t query = valid ? first + column : begins;
        const uint32_t node = nodes.from + query / a.group, head = h * a.group + query % a.group;
        Query<S::kType, HD> q;
        q.fetch(a.query + node * a.query_stride + size_t(head) * kv.head_dim, valid, kv.head_dim,
                lane);
        const uint32_t *mask = a.d.mask + node * a.d.mask_stride;
        const uint32_t words = (nodes.count + 31) / 32;
        q.convert(a.scale);

        Softmax<S::kType, HD> sm;
        // a thread's chunks of the next stage of fp32 rows
        constexpr int kHeld = TYPE == NUT_F32 ? (kWork == 0 ? 1 : kWork) : 1;
        float ahead[2][kHeld][8];

        // Where the segment's rows lie, kPiece at a time, a thread a row: the table is
        // asked for a piece while the one before it is multiplied, by DMA, as a load into
        // registers would have to be waited for, and all that was asked for before it.
        const auto ask_table = [&](uint32_t piece) {
            const uint32_t index = page_of(kv, begin + piece * kPiece) + threadIdx.x;
            if (threadIdx.x < kPiece && index <= page_of(kv, begin + count - 1))
                stage_dma<4>(a.s.table + size_t(b) * a.s.table_stride + index,
                             table + wave * kWave);
        };
        const auto place_rows = [&](uint32_t piece) {
            const uint32_t i = piece * kPiece + threadIdx.x, row = begin + i;
            size_t at = kNoRow;
            if (threadIdx.x >= kPiece) // whole waves
                return;
            if (i < count) {
                const uint32_t index = page_of(kv, row);
                const int page = table[index - page_of(kv, row - threadIdx.x)];
                if (page_in(page, kv.pages))
                    at = size_t(page) * kv.page_stride + h * kv.head_stride +
                         (row - index * kv.page_size) * kv.slot_stride;
                else
                    status_flag(kv.status, kBadPage);
            }
            offsets[piece % 2][threadIdx.x] = at;
            const uint64_t masked = __ballot(at == kNoRow);
            if (lane % 32 == 0)
                gone[piece % 2][threadIdx.x / 32] = uint32_t(masked >> lane);
        };
        const auto offset_of = [&](uint32_t s) { return offsets[s / kEach % 2] + s % kEach * R; };
        const auto gone_of = [&](uint32_t s, int half) {
            return gone[s / kEach % 2][s % kEach * (R / 32) + half];
        };
        // Whether there are rows behind the piece of stage s.
        const auto more = [&](uint32_t s) { return (s / kEach + 1) * kPiece < count; };
        static_assert(kEach > S::kBuffers, "a piece is placed before its first stage is fetched");
        const uint32_t stages = (count + R - 1) / R;
        // Chunk i of a stage: row i / kChunks, as place() lays them. Rows that are none
        // are zeros.
        const auto fetch = [&](uint32_t s) {
            const size_t *rows = offset_of(s);
            if constexpr (TYPE == NUT_F32) {
#pragma unroll
                for (int w = 0; w < kHeld; w++) {
                    const uint32_t i = w * 256 + threadIdx.x, row = i / S::kChunks;
                    const uint32_t chunk = i % S::kChunks;
                    // without a branch, so that the chunks stay in registers
                    const size_t at = row < uint32_t(R) ? rows[row] : kNoRow;
                    const bool there = at != kNoRow && chunk < used;
                    const size_t byte = there ? at + chunk * 32 : 0;
                    load8<NUT_F32>(kv.keys + byte, ahead[0][w]);
                    load8<NUT_F32>(kv.values + byte, ahead[1][w]);
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            ahead[x][w][e] = there ? ahead[x][w][e] : 0.0f;
                }
            } else {
                char *keys = stage[s % S::kBuffers][0], *values = stage[s % S::kBuffers][1];
                for (uint32_t i = wave * kWave; i < uint32_t(R) * S::kChunks; i += 256) {
                    const uint32_t from = S::place(i + lane), row = from / S::kChunks;
                    const uint32_t chunk = from % S::kChunks;
                    const size_t at = rows[row];
                    if (chunk < used && at != kNoRow && a.past) {
                        stage_dma<16, true>(kv.keys + at + chunk * 16, keys + i * 16);
                        stage_dma<16, true>(kv.values + at + chunk * 16, values + i * 16);
                    } else if (chunk < used && at != kNoRow) {
                        stage_dma(kv.keys + at + chunk * 16, keys + i * 16);
                        stage_dma(kv.values + at + chunk * 16, values + i * 16);
                    } else if (chunk < used) {
                        const u32x4 zero{0, 0, 0, 0};
                        *reinterpret_cast<u32x4 *>(keys + (i + lane) * 16) = zero;
                        *reinterpret_cast<u32x4 *>(values + (i + lane) * 16) = zero;
                    }
                }
            }
        };
        __syncthreads(); // the segment before is done with
        if (stages != 0)
            ask_table(0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        place_rows(0);
        __syncthreads();
        if (stages != 0)
            fetch(0);
        for (uint32_t s = 0; s < stages; s++) {
            char *keys = stage[s % S::kBuffers][0], *values = stage[s % S::kBuffers][1];
            uint32_t *odd_rows = strange[s % 2]; // the other stage's may still be read
            const uint32_t row = begin + s * R;
            const bool drafted = row + R > held;
            if constexpr (TYPE == NUT_F32) {
                if (s != 0)
                    __syncthreads(); // the stage before is done with
                if (threadIdx.x < 2)
                    odd_rows[threadIdx.x] = 0;
                if (drafted)
                    __syncthreads();
#pragma unroll
                for (int w = 0; w < kHeld; w++) {
                    const uint32_t i = w * 256 + threadIdx.x, own = i / S::kChunks;
                    const bool there = kWork != 0 || own < uint32_t(R);
                    if (drafted) { // values that are not finite are added one by one
                        bool odd = false;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const bool is = !(fabsf(ahead[1][w][e]) < INFINITY);
                            odd = odd || is;
                            ahead[1][w][e] = is ? 0.0f : ahead[1][w][e];
                        }
                        if (odd && there)
                            atomicOr(&odd_rows[own / 32], 1u << (own % 32));
                    }
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        u32x4 limb[3];
                        split<NUT_BF16, 3>(ahead[x][w], limb);
                        if (there)
#pragma unroll
                            for (int p = 0; p < 3; p++)
                                *reinterpret_cast<u32x4 *>(
                                    (x == 0 ? keys : values) +
                                    S::place(p * R * S::kChunks + i) * 16) = limb[p];
                    }
                }
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // a table that was asked for
                __syncthreads();
                if (s % kEach == 0 && more(s))
                    ask_table(s / kEach + 1);
                if (s % kEach == 1 && more(s))
                    place_rows(s / kEach + 1);
                if (s + 1 < stages)
                    fetch(s + 1);
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                if (drafted && threadIdx.x < 2)
                    odd_rows[threadIdx.x] = 0;
                __syncthreads(); // the stage is there, the one before done with
                if (s % kEach == 0 && more(s)) // older than the stage that follows it
                    ask_table(s / kEach + 1);
                if (s % kEach == 1 && more(s)) // first read one barrier from here
                    place_rows(s / kEach + 1);
                if (s + 1 < stages)
                    fetch(s + 1);
                if (drafted) {
                    for (uint32_t i = threadIdx.x; i < uint32_t(R) * S::kChunks; i += 256) {
                        const uint32_t from = S::place(i), own = from / S::kChunks;
                        if (from % S::kChunks >= used) // no chunk of a row: never written
                            continue;
                        u32x4 *v = reinterpret_cast<u32x4 *>(values + i * 16);
                        u32x4 x = *v;
                        bool odd = false;
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            constexpr uint32_t e = TYPE == NUT_F16 ? 0x7c00u : 0x7f80u;
                            const bool lo = (x[w] & e) == e, hi = (x[w] >> 16 & e) == e;
                            odd = odd || lo || hi;
                            x[w] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
                        }
                        if (odd) {
                            *v = x;
                            atomicOr(&odd_rows[own / 32], 1u << (own % 32));
                        }
                    }
                    __syncthreads();
                }
            }
            if (first >= queries)
                continue;
            constexpr int kHalves = R / 32;
            uint32_t none[kHalves], odd[kHalves], seen[kHalves];
#pragma unroll
            for (int half = 0; half < kHalves; half++) {
                none[half] = uint32_t(__builtin_amdgcn_readfirstlane(gone_of(s, half)));
                odd[half] = drafted ? uint32_t(__builtin_amdgcn_readfirstlane(odd_rows[half])) &
                                          ~none[half]
                                    : 0;
                seen[half] = !drafted ? ~0u
                                      : mask_bits(int64_t(row + half * 32) - held, words,
                                                  [&](uint32_t w) { return mask[w]; });
            }
            attend_stage<TYPE, HD, FULL>(keys, values, offset_of(s), none, drafted, odd, seen, q,
                                         sm, kv, lane);
        }

        float sum = sm.sum;
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (!valid)
            continue;
        const size_t at = size_t(node) * a.heads + head;
        const size_t part = size_t(slot) * kBlock + (query - begins);
        const float f = cut ? 1.0f : 1.0f / sum;
        float *to = cut ? a.parts + part * kv.head_dim : a.out + at * kv.head_dim;
#pragma unroll
        for (int g = 0; g < G; g++)
            if (FULL || 16 * g + 4 * j < kv.head_dim)
                *reinterpret_cast<f32x4 *>(to + 16 * g + 4 * j) =
                    !cut && sum == 0.0f ? f32x4{0, 0, 0, 0} : sm.o[g] * f;
        if (j == 0 && cut)
            a.stats[part] = make_float2(sum == 0.0f ? -INFINITY : sm.ref, sum);
        if (j == 0 && !cut && a.lse != nullptr)
            a.lse[at] = sum == 0.0f ? -INFINITY
                                    : (sm.ref + log2f(sum)) * 0.69314718055994531f;
    }
}

// Sums of a query row's parts, four components of it.
struct Joined {
    float most, sum;
    f32x4 o;
};

// Parts `first`, first + step, .. below `end`, whose exponents and sums are at stat(r)
// and components at part(r); kAtOnce loads in flight together.
template <typename Stat, typename Part>
__device__ __forceinline__ Joined join_parts(uint32_t first, uint32_t step, uint32_t end,
                                             Stat &&stat, Part &&part)
{
    constexpr int kAtOnce = 8;
    Joined to{-INFINITY, 0.0f, f32x4{0, 0, 0, 0}};
    for (uint32_t r = first; r < end; r += kAtOnce * step) {
        float2 st[kAtOnce];
        f32x4 x[kAtOnce];
#pragma unroll
        for (int e = 0; e < kAtOnce; e++) { // behind the last: the last again, without weight
            const uint32_t own = min(r + e * step, end - 1);
            st[e] = *stat(own);
            x[e] = *part(own);
        }
        float now = to.most;
#pragma unroll
        for (int e = 0; e < kAtOnce; e++)
            now = r + e * step < end ? fmaxf(now, st[e].x) : now;
        if (now == -INFINITY)
            continue;
        const float f = to.most == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(to.most - now);
        to.sum *= f;
        to.o *= f;
        to.most = now;
#pragma unroll
        for (int e = 0; e < kAtOnce; e++) {
            if (r + e * step >= end || st[e].x == -INFINITY) // no row of a finite score: not summed
                continue;
            const float g = __builtin_amdgcn_exp2f(st[e].x - now);
            to.sum = fmaf(st[e].y, g, to.sum);
#pragma unroll
            for (int d = 0; d < 4; d++)
                to.o[d] = fmaf(x[e][d], g, to.o[d]);
        }
    }
    return to;
}

// A workgroup of the joins: threads of `teams` teams to a query row, each a part of the
// row's parts in turn, tpr threads to a team.
struct Team {
    uint32_t row, team, part;
    bool in;
};
__device__ __forceinline__ Team team_of(uint32_t teams, uint32_t tpr)
{
    const uint32_t all = threadIdx.x / tpr;
    return Team{all / teams, all % teams, threadIdx.x - all * tpr, all < 256 / tpr / teams * teams};
}

// What a query row's teams have summed, written by its first one.
__device__ __forceinline__ void write_joined(const TreeArgs &a, const Team &t, uint32_t teams,
                                             uint32_t tpr, Joined own, size_t at, bool valid)
{
    __shared__ Joined others[256];
    if (teams > 1) {
        others[threadIdx.x] = own;
        __syncthreads();
        if (t.team == 0 && valid)
            own = join_parts(
                0, 1, teams,
                [&](uint32_t r) {
                    return reinterpret_cast<const float2 *>(&others[threadIdx.x + r * tpr].most);
                },
                [&](uint32_t r) { return &others[threadIdx.x + r * tpr].o; });
    }
    if (!valid || t.team != 0)
        return;
    const float f = own.sum == 0.0f ? 0.0f : 1.0f / own.sum;
    *reinterpret_cast<f32x4 *>(a.out + at * a.kv.head_dim + t.part * 4) = own.o * f;
    if (t.part == 0 && a.lse != nullptr)
        a.lse[at] = own.sum == 0.0f ? -INFINITY
                                    : (own.most + log2f(own.sum)) * 0.69314718055994531f;
}

// The shares of an item joined, where it was cut; a team takes every a.teams-th of them.
template <int R>
__global__ __launch_bounds__(256) void staged_join_kernel(TreeArgs a)
{
    const uint32_t tpr = a.kv.head_dim / 4, rows = 256 / tpr / a.teams; // of a workgroup
    const uint32_t groups = (kBlock + rows - 1) / rows;
    const uint32_t b = blockIdx.y, item = blockIdx.x / groups;
    const uint64_t start = a.before[b], all = a.before[a.s.batch];
    const Item it = item_of<R>(a, b, false);
    const uint32_t h = it.blocks == 0 ? 0 : item / it.blocks;
    if (it.blocks == 0 || h >= a.kv.kv_heads)
        return;
    const Shares shares{all, share_count(all, a.shares)};
    const uint64_t begin = start + uint64_t(item) * it.stages;
    const uint32_t first = shares.of(begin), last = shares.of(begin + it.stages - 1);
    if (first == last)
        return;
    const uint32_t begins = (item - h * it.blocks) * kBlock;
    const uint32_t queries = min(kBlock, it.nodes.count * a.group - begins);
    const Team t = team_of(a.teams, tpr);
    const uint32_t k = (blockIdx.x - item * groups) * rows + t.row, row = begins + k;
    const bool valid = t.in && k < queries;
    // a share's second slot is of the item that it ends in
    const auto slot = [&](uint32_t share) {
        return size_t(2 * share + (share == first)) * kBlock + k;
    };
    Joined own{-INFINITY, 0.0f, f32x4{0, 0, 0, 0}};
    if (valid)
        own = join_parts(
            first + t.team, a.teams, last + 1, [&](uint32_t r) { return a.stats + slot(r); },
            [&](uint32_t r) {
                return reinterpret_cast<const f32x4 *>(a.parts) + slot(r) * tpr + t.part;
            });
    write_joined(a, t, a.teams, tpr, own,
                 size_t(it.nodes.from + row / a.group) * a.heads + h * a.group + row % a.group,
                 valid);
}

// The runs joined.
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a)
{
    const uint32_t b = blockIdx.y, tpr = a.kv.head_dim / 4, rows = 256 / tpr / a.teams;
    const NodeSpan nodes = nodes_of(a.d, b, false);
    const uint64_t all = uint64_t(nodes.count) * a.heads;
    if (uint64_t(blockIdx.x) * rows >= all)
        return;
    uint32_t held;
    const uint32_t total = rows_of(a, b, nodes.count, held, false);
    const uint32_t runs = (total + a.run - 1) / a.run;
    const Team t = team_of(a.teams, tpr);
    const uint64_t row = uint64_t(blockIdx.x) * rows + t.row;
    const bool valid = t.in && row < all;
    const size_t at = size_t(nodes.from) * a.heads + row;
    Joined own{-INFINITY, 0.0f, f32x4{0, 0, 0, 0}};
    if (valid)
        own = join_parts(
            t.team, a.teams, runs, [&](uint32_t r) { return a.stats + at * a.runs + r; },
            [&](uint32_t r) {
                return reinterpret_cast<const f32x4 *>(a.parts) + (at * a.runs + r) * tpr + t.part;
            });
    write_joined(a, t, a.teams, tpr, own, at, valid);
}

template <int TYPE, int HD, int WQ>
void tree_by(const TreeArgs &a, dim3 grid, hipStream_t stream)
{
    const auto run = a.kv.head_dim == HD ? tree_kernel<TYPE, HD, true, WQ>
                                         : tree_kernel<TYPE, HD, false, WQ>;
    hipLaunchKernelGGL(run, grid, dim3(64 * kTreeWaves<HD>), 0, stream, a);
}

template <int TYPE, int HD>
void tree_as(const TreeArgs &a, const TreePlan &plan, dim3 grid, hipStream_t stream)
{
    const bool full = a.kv.head_dim == HD;
    if (plan.staged) {
        const auto run = full ? staged_kernel<TYPE, HD, true> : staged_kernel<TYPE, HD, false>;
        const auto join = staged_join_kernel<Stage<TYPE, HD>::kRows>;
        hipLaunchKernelGGL(run, dim3(plan.shares), dim3(256), 0, stream, a);
        check_launch("tree attention");
        hipLaunchKernelGGL(join, grid, dim3(256), 0, stream, a);
    } else if (plan.waves == 1) {
        tree_by<TYPE, HD, 1>(a, grid, stream);
    } else {
        tree_by<TYPE, HD, 2>(a, grid, stream);
    }
}

template <int TYPE>
void tree_in(const TreeArgs &a, const TreePlan &plan, dim3 grid, hipStream_t stream)
{
    if (a.kv.head_dim <= 32)
        tree_as<TYPE, 32>(a, plan, grid, stream);
    else if (a.kv.head_dim <= 64)
        tree_as<TYPE, 64>(a, plan, grid, stream);
    else if (a.kv.head_dim <= 96)
        tree_as<TYPE, 96>(a, plan, grid, stream);
    else if (a.kv.head_dim <= 128)
        tree_as<TYPE, 128>(a, plan, grid, stream);
    else
        tree_as<TYPE, 256>(a, plan, grid, stream);
}

// Teams that join a query row of so many parts, eight in flight a team. (Two sequences of
// 14,283 to 17,791 fp32 rows, 3 KV heads of 80, 3 nodes, 140 runs: the call 139 us where
// one thread went from run to run, 37 with teams.)
uint32_t teams_for(const PagedView &kv, uint64_t parts)
{
    uint32_t teams = 1;
    while (teams * 8 < parts && teams * 2 * (kv.head_dim / 4) <= 256)
        teams *= 2;
    return teams;
}
// Query rows of a workgroup of the join.
uint32_t joined_rows(const PagedView &kv, const TreePlan &plan)
{
    return 256 / (kv.head_dim / 4) / plan.teams;
}

} // namespace

TreePlan plan_tree(const PagedView &kv, const PagedSeqs &seqs, const DraftView &draft,
                   uint32_t heads)
{
    const auto aligned = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
    TreePlan plan{};
    const uint64_t queries = uint64_t(draft.most) * (heads / kv.kv_heads);
    require(queries * kv.kv_heads <= 0x7fffffff, NUT_EINVAL,
            "paged cache: more rows than one launch covers");
    // Rows in shared memory pay for sharing out and joining; from 33 query rows a KV head
    // on, where 16 of them and 128 rows of a sequence make more than 1,024 workgroups.
    // tree_kernel and staged_kernel, us, 32 heads of 64 on 4 KV heads. 64 nodes: 16
    // sequences of 2,000 bfloat16 rows 83 and 57, of 1,000 48 and 43, fp32 146 and 86, 81
    // and 56; below the bound one of 700 13.8 and 19.0, fp32 16.6 and 20.8. Just above it
    // 16-bit rows lose: 16 of 500 31 and 34, of 100 17 and 26. 8 nodes: 64 of 8,000 222
    // and 135, of 1,000 32 and 34, of 200 13 and 21. 4 nodes, 32 query rows: 16 of 4,000
    // to 8,192 38.6 and 41, though 64 of them 128 and 99.
    const uint64_t small = uint64_t(draft.batch) * kv.kv_heads * ((queries + 15) / 16) *
                           ((seqs.max_length + 127) / 128);
    plan.staged = queries > 32 && small > 1024;
    if (plan.staged) {
        // as many workgroups as the chip holds at once, by registers and shared memory
        plan.shares = 256 * staged_groups(kv.type, kv.head_dim);
        plan.blocks = uint32_t((queries + kBlock - 1) / kBlock);
        // 16-bit rows that are read once, and are more than the caches hold: nothing of
        // them is there when the next call comes. Through the caches and past them, us,
        // 64 nodes of 32 fp16 heads of 128: 32 MiB 34 and 36, 64 44 and 45, 128 59 and 57,
        // 512 150 and 143, 2,044 459 and 444.
        const uint64_t bytes = uint64_t(seqs.max_length) * draft.batch * kv.kv_heads *
                               kv.head_dim * 2 * paged_element(kv.type);
        plan.past = kv.type != NUT_F32 && plan.blocks == 1 && bytes >= (128ull << 20);
        // in the mean, where lengths differ
        plan.teams =
            teams_for(kv, plan.shares / (uint64_t(draft.batch) * kv.kv_heads * plan.blocks) + 1);
        require(draft.batch <= 65535, NUT_EINVAL, "paged cache: more rows than one launch covers");
        paged_grid(uint64_t(draft.batch) * kv.kv_heads * plan.blocks * kBlock, 256);
        plan.stats = aligned(size_t(plan.shares) * 2 * kBlock * kv.head_dim * sizeof(float));
        plan.before = plan.stats + aligned(size_t(plan.shares) * 2 * kBlock * sizeof(float2));
        plan.bytes = plan.before + aligned((size_t(draft.batch) + 1) * sizeof(uint64_t));
        return plan;
    }
    // Two tiles of query rows read a sequence once for both. One and two, us: 27 nodes of
    // 32 fp16 heads of 128, 32 sequences of 10 to 64 rows 36 and 24, 4 of 8,000 to 16,000
    // 234 and 193, though 16 of 500 to 2,048 99 and 104; 4 nodes of 8 heads of 64 a KV
    // head, 16 of 4,000 to 8,192 bfloat16 rows 44 and 39, of 100 to 512 13.3 and 14.3.
    plan.waves = queries > 16 && small > 1024 ? 2 : 1;
    plan.blocks = uint32_t((queries + 16 * plan.waves - 1) / (16 * plan.waves));
    const uint64_t columns = uint64_t(draft.batch) * kv.kv_heads * plan.blocks;
    // Runs as long as make 1,024 workgroups, or down to 128 rows.
    plan.run = (seqs.max_length + 127) / 128 * 128;
    while (plan.run > 128 && columns * ((seqs.max_length + plan.run - 1) / plan.run) < 1024)
        plan.run = (plan.run / 2 + 127) / 128 * 128;
    plan.runs = (seqs.max_length + plan.run - 1) / plan.run;
    const uint64_t units = uint64_t(draft.batch) * kv.kv_heads * plan.runs;
    paged_grid((units + 7) / 8 * 8 * plan.blocks, 256);
    if (plan.runs == 1)
        return plan;
    plan.teams = teams_for(kv, plan.runs);
    const uint32_t joined = joined_rows(kv, plan);
    paged_grid((uint64_t(draft.most) * heads + joined - 1) / joined, 256);
    require(draft.batch <= 65535, NUT_EINVAL, "paged cache: more rows than one launch covers");
    const size_t parts = size_t(draft.total) * heads * plan.runs;
    plan.stats = aligned(parts * kv.head_dim * sizeof(float));
    plan.bytes = plan.stats + aligned(parts * sizeof(float2));
    return plan;
}

void launch_tree_attention(const PagedView &kv, const PagedSeqs &seqs, const DraftView &draft,
                           const float *query, size_t query_stride, uint32_t heads, float scale,
                           float *out, float *lse, char *workspace, hipStream_t stream)
{
    const TreePlan plan = plan_tree(kv, seqs, draft, heads);
    const uint64_t units = uint64_t(draft.batch) * kv.kv_heads * plan.runs;
    TreeArgs a{kv, seqs, draft, query, query_stride, heads, heads / kv.kv_heads,
               scale * 1.4426950408889634f, out, lse, plan.blocks, plan.run, plan.runs,
               uint32_t(units), plan.shares, plan.teams, plan.past, nullptr, nullptr, nullptr};
    if (plan.bytes != 0) {
        a.parts = reinterpret_cast<float *>(workspace);
        a.stats = reinterpret_cast<float2 *>(workspace + plan.stats);
        a.before = reinterpret_cast<uint64_t *>(workspace + plan.before);
    }
    const uint32_t joined = plan.teams == 0 ? 1 : joined_rows(kv, plan);
    const uint32_t groups = (kBlock + joined - 1) / joined; // workgroups of the join, an item
    const dim3 grid = plan.staged ? dim3(kv.kv_heads * plan.blocks * groups, draft.batch)
                                  : paged_grid((units + 7) / 8 * 8 * plan.blocks, 256);
    if (kv.type == NUT_F32)
        tree_in<NUT_F32>(a, plan, grid, stream);
    else if (kv.type == NUT_F16)
        tree_in<NUT_F16>(a, plan, grid, stream);
    else
        tree_in<NUT_BF16>(a, plan, grid, stream);
    check_launch("tree attention");
    if (plan.staged || plan.runs == 1)
        return;
    const uint64_t rows = uint64_t(draft.most) * heads;
    hipLaunchKernelGGL(tree_join_kernel, dim3(uint32_t((rows + joined - 1) / joined), draft.batch),
                       dim3(256), 0, stream, a);
    check_launch("tree attention");
}

} // namespace nut
