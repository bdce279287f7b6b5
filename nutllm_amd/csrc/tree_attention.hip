// tree_attention.hip — attention of a tree of drafted tokens over a paged KV
// cache.
//
// The query rows of a KV head are its sequence's nodes times the heads that
// share it, node after node. A workgroup takes a block of them and a run of the
// sequence's rows; its waves take tiles of the run in turn, as in
// paged_attention.hip, but multiply a tile in registers with QT tiles of 16
// query rows, not one. Rows that the sequence held before are seen by every node;
// of a tile that reaches into the drafted rows each lane takes its node's mask.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "paged_attend.hpp"
#include "runtime.hpp"
#include "serving.hpp"

namespace nut {

namespace {

constexpr uint32_t kPiece = 1024; // rows whose offsets are in shared memory at once

struct TreeArgs {
    PagedView kv;
    PagedSeqs s;
    DraftView d;
    const float *query;
    size_t query_stride;
    uint32_t heads, group;
    float scale; // times log2(e)
    float *out, *lse;
    uint32_t blocks, run, runs, units;
    float *parts;  // [total][heads][runs][head_dim], unnormalised
    float2 *stats; // [total][heads][runs]: exponent they refer to, sum
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

// A tile against QT tiles of query rows. `gone`: rows that no node sees, the
// same in every lane; `seen`: with `drafted`, the rows that the lane's node of
// each query tile sees.
template <int TYPE, int HD, bool FULL, int QT>
__device__ __forceinline__ void attend_tree(Tile<TYPE, HD> &tile, const size_t *at, uint32_t gone,
                                            bool drafted, const uint32_t (&seen)[QT],
                                            const Query<TYPE, HD> (&q)[QT],
                                            Softmax<TYPE, HD> (&sm)[QT], const PagedView &kv,
                                            int lane)
{
    using T = Tile<TYPE, HD>;
    constexpr int G = T::G, E = T::kEach;
    const int j = lane >> 4;
    float s[QT][T::kScores];
#pragma unroll
    for (int t = 0; t < QT; t++)
        score<TYPE, HD>(tile, q[t], s[t]);
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
#pragma unroll
            for (int t = 0; t < QT; t++)
                s[t][r] = out || !(seen[t] >> (4 * j) >> bit & 1) ? -INFINITY : s[t][r];
            if (drafted) {
                const uint64_t any = __ballot(strange);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    odd |= (any >> (16 * i) & 0xffff) != 0 ? 1u << (bit + 4 * i) : 0;
            }
        }
        odd = __builtin_amdgcn_readfirstlane(odd);
    }
    float p[QT][8];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        float most = s[t][0];
#pragma unroll
        for (int r = 1; r < T::kScores; r++)
            most = fmaxf(most, s[t][r]);
        sm[t].raise(max_over_rows(most));
#pragma unroll
        for (int r = 0; r < T::kScores; r++) {
            p[t][r] = __builtin_amdgcn_exp2f(s[t][r] - sm[t].ref);
            sm[t].sum += p[t][r];
        }
    }
    if (odd != 0) {
        // 0 times what is not finite is no number: such rows leave the product,
        // and nodes that weigh them add them one by one.
        for (uint32_t left = odd; left != 0; left &= left - 1) {
            const int row = __builtin_ctz(left), own = row % 16 / 4;
            const char *v = kv.values + at[row];
#pragma unroll
            for (int t = 0; t < QT; t++) {
                float weight = 0.0f;
#pragma unroll
                for (int r = 0; r < T::kScores; r++)
                    if (16 * (r / 4) + r % 4 == row - 4 * own)
                        weight = p[t][r];
                weight = __shfl(weight, 16 * own + (lane & 15));
#pragma unroll
                for (int g = 0; g < G; g++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t d = 16 * (g / E * E) + 4 * j * E + i * E + g % E;
                        if (weight != 0.0f && (FULL || d < kv.head_dim))
                            sm[t].o[g][i] = fmaf(weight, component<TYPE>(v, d), sm[t].o[g][i]);
                    }
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
#pragma unroll
                for (int t = 0; t < QT; t++)
                    sm[t].o[g] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                        __uint_as_float(tile.v[r][g]), p[t][r], sm[t].o[g], 0, 0, 0);
    } else {
        constexpr int kLimbs = Query<TYPE, HD>::kLimbs;
        u32x4 limb[QT][kLimbs];
#pragma unroll
        for (int t = 0; t < QT; t++)
            split<TYPE, kLimbs>(p[t], limb[t]);
#pragma unroll
        for (int g = 0; g < G; g++) {
            const u32x4 x = tile.component(g);
#pragma unroll
            for (int l = kLimbs - 1; l >= 0; l--)
#pragma unroll
                for (int t = 0; t < QT; t++)
                    sm[t].o[g] = product<TYPE>(x, limb[t][l], sm[t].o[g]);
        }
    }
}

template <int HD> constexpr int kTreeWaves = HD == 256 ? 2 : 4;

template <int TYPE, int HD, bool FULL, int QT>
__global__ __launch_bounds__(64 * kTreeWaves<HD>, HD == 256 ? 1 : 2) void tree_kernel(TreeArgs a)
{
    using T = Tile<TYPE, HD>;
    constexpr int G = T::G, WAVES = kTreeWaves<HD>, kThreads = 64 * WAVES;
    constexpr int kStride = HD + 4;
    __shared__ union Shared {
        size_t at[kPiece];
        float o[WAVES][16][kStride];
    } lds;
    __shared__ float stat[3][WAVES][16];
    __shared__ uint32_t gone[kPiece / 32];
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
    const uint32_t queries = nodes.count * a.group, first = block * QT * 16;
    if (first >= queries)
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
    Query<TYPE, HD> q[QT];
    const uint32_t *mask[QT];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const uint32_t row = first + t * 16 + column;
        const bool valid = row < queries;
        const uint32_t node = nodes.from + (valid ? row : first) / a.group;
        const uint32_t head = h * a.group + (valid ? row : first) % a.group;
        q[t].fetch(a.query + node * a.query_stride + size_t(head) * kv.head_dim, valid,
                   kv.head_dim, lane);
        mask[t] = a.d.mask + node * a.d.mask_stride;
    }
    const uint32_t words = (nodes.count + 31) / 32;
#pragma unroll
    for (int t = 0; t < QT; t++)
        q[t].convert(a.scale);

    Softmax<TYPE, HD> sm[QT];
    for (uint32_t piece = 0; piece < count; piece += kPiece) {
        const uint32_t rows = min(count - piece, kPiece);
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
        const int tiles = int((rows + T::kRows - 1) / T::kRows);
        for (int t = wave; t < tiles; t += WAVES) {
            Tile<TYPE, HD> x;
            x.template load<FULL, false>(kv, lds.at + t * T::kRows, lane);
            const uint32_t none = uint32_t(__builtin_amdgcn_readfirstlane(
                gone[t * T::kRows / 32] >> (t * T::kRows % 32) & kAll));
            const uint32_t row = begin + piece + t * T::kRows;
            const bool drafted = row + T::kRows > held;
            uint32_t seen[QT];
#pragma unroll
            for (int k = 0; k < QT; k++)
                seen[k] = !drafted ? ~0u
                                   : mask_bits(int64_t(row) - held, words,
                                               [&](uint32_t w) { return mask[k][w]; });
            attend_tree<TYPE, HD, FULL, QT>(x, lds.at + t * T::kRows, none, drafted, seen, q, sm,
                                            kv, lane);
        }
    }

    // The waves' sums side by side, a tile of query rows at a time; then a thread
    // per four components adds them.
    const uint32_t parts = FULL ? HD / 4 : kv.head_dim / 4;
#pragma unroll
    for (int t = 0; t < QT; t++) {
        if (first + t * 16 >= queries)
            break;
        sm[t].sum += __shfl_xor(sm[t].sum, 16);
        sm[t].sum += __shfl_xor(sm[t].sum, 32);
        __syncthreads();
        if (j == 0)
            stat[0][wave][column] = sm[t].most, stat[1][wave][column] = sm[t].ref,
            stat[2][wave][column] = sm[t].sum;
        constexpr int E = T::kEach;
#pragma unroll
        for (int p = 0; p < G; p += E) {
            float flat[4 * E]; // components 16 p + 4 j E .. of the lane's query row
#pragma unroll
            for (int g = 0; g < E; g++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    flat[i * E + g] = sm[t].o[p + g][i];
            float *to = lds.o[wave][column] + 16 * p + 4 * j * E;
#pragma unroll
            for (int d = 0; d < 4 * E; d += 4)
                *reinterpret_cast<f32x4 *>(to + d) =
                    f32x4{flat[d], flat[d + 1], flat[d + 2], flat[d + 3]};
        }
        __syncthreads();
        const uint32_t here = min(16u, queries - first - t * 16);
        for (uint32_t i = threadIdx.x; i < here * parts; i += kThreads) {
            const uint32_t k = i / parts, d = i % parts * 4;
            float most = stat[0][0][k];
#pragma unroll
            for (int w = 1; w < WAVES; w++)
                most = fmaxf(most, stat[0][w][k]);
            const float ref = most == -INFINITY ? 0.0f : most - Softmax<TYPE, HD>::kShift;
            float sum = 0.0f;
            f32x4 o{0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                // what no row of a finite score reached is zero, or not a number
                const float f = stat[0][w][k] == -INFINITY
                                    ? 1.0f
                                    : __builtin_amdgcn_exp2f(stat[1][w][k] - ref);
                sum = fmaf(stat[2][w][k], f, sum);
                const f32x4 y = *reinterpret_cast<const f32x4 *>(&lds.o[w][k][d]);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    o[e] = fmaf(y[e], f, o[e]);
            }
            const uint32_t row = first + t * 16 + k;
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
}

// The runs joined: a thread for four components of a node's head.
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a)
{
    const uint32_t b = blockIdx.y, tpr = a.kv.head_dim / 4;
    const NodeSpan nodes = nodes_of(a.d, b, false);
    const uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    const uint64_t row = i / tpr;
    if (row >= uint64_t(nodes.count) * a.heads)
        return;
    uint32_t held;
    const uint32_t total = rows_of(a, b, nodes.count, held, false);
    const uint32_t runs = (total + a.run - 1) / a.run, part = uint32_t(i - row * tpr);
    const size_t at = size_t(nodes.from) * a.heads + row;
    const float2 *stats = a.stats + at * a.runs;
    const f32x4 *parts =
        reinterpret_cast<const f32x4 *>(a.parts + at * a.runs * a.kv.head_dim) + part;
    float most = -INFINITY;
    for (uint32_t r = 0; r < runs; r++)
        most = fmaxf(most, stats[r].x);
    float sum = 0.0f;
    f32x4 o{0, 0, 0, 0};
    for (uint32_t r = 0; r < runs; r++) {
        const float2 st = stats[r];
        const f32x4 x = parts[r * tpr];
        if (st.x == -INFINITY) // no row of a finite score: not summed
            continue;
        const float f = __builtin_amdgcn_exp2f(st.x - most);
        sum = fmaf(st.y, f, sum);
#pragma unroll
        for (int e = 0; e < 4; e++)
            o[e] = fmaf(x[e], f, o[e]);
    }
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    *reinterpret_cast<f32x4 *>(a.out + at * a.kv.head_dim + part * 4) = o * f;
    if (part == 0 && a.lse != nullptr)
        a.lse[at] = sum == 0.0f ? -INFINITY : (most + log2f(sum)) * 0.69314718055994531f;
}

// Query tiles of a block at most, by what fits the registers of two waves a SIMD.
constexpr uint32_t most_queries(uint32_t head_dim)
{
    return head_dim <= 64 ? 4 : head_dim <= 128 ? 2 : 1;
}

template <int TYPE, int HD>
void tree_as(const TreeArgs &a, uint32_t queries, dim3 grid, hipStream_t stream)
{
    const bool full = a.kv.head_dim == HD;
    auto run = full ? tree_kernel<TYPE, HD, true, 1> : tree_kernel<TYPE, HD, false, 1>;
    if constexpr (most_queries(HD) >= 2)
        if (queries == 2)
            run = full ? tree_kernel<TYPE, HD, true, 2> : tree_kernel<TYPE, HD, false, 2>;
    if constexpr (most_queries(HD) >= 4)
        if (queries == 4)
            run = full ? tree_kernel<TYPE, HD, true, 4> : tree_kernel<TYPE, HD, false, 4>;
    hipLaunchKernelGGL(run, grid, dim3(64 * kTreeWaves<HD>), 0, stream, a);
}

template <int TYPE>
void tree_in(const TreeArgs &a, uint32_t queries, dim3 grid, hipStream_t stream)
{
    if (a.kv.head_dim <= 32)
        tree_as<TYPE, 32>(a, queries, grid, stream);
    else if (a.kv.head_dim <= 64)
        tree_as<TYPE, 64>(a, queries, grid, stream);
    else if (a.kv.head_dim <= 96)
        tree_as<TYPE, 96>(a, queries, grid, stream);
    else if (a.kv.head_dim <= 128)
        tree_as<TYPE, 128>(a, queries, grid, stream);
    else
        tree_as<TYPE, 256>(a, queries, grid, stream);
}

} // namespace

TreePlan plan_tree(const PagedView &kv, const PagedSeqs &seqs, const DraftView &draft,
                   uint32_t heads)
{
    const auto aligned = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
    TreePlan plan{};
    const uint64_t queries = uint64_t(draft.most) * (heads / kv.kv_heads);
    require(queries <= 0x7fffffff, NUT_EINVAL, "paged cache: more rows than one launch covers");
    plan.queries = 1;
    while (plan.queries < most_queries(kv.head_dim) && plan.queries * 16 < queries)
        plan.queries *= 2;
    plan.blocks = uint32_t((queries + plan.queries * 16 - 1) / (plan.queries * 16));
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
    paged_grid((uint64_t(draft.most) * heads * (kv.head_dim / 4) + 255) / 256 * 256, 1);
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
               uint32_t(units), nullptr, nullptr};
    if (plan.runs > 1) {
        a.parts = reinterpret_cast<float *>(workspace);
        a.stats = reinterpret_cast<float2 *>(workspace + plan.stats);
    }
    const dim3 grid = paged_grid((units + 7) / 8 * 8 * plan.blocks, 256);
    if (kv.type == NUT_F32)
        tree_in<NUT_F32>(a, plan.queries, grid, stream);
    else if (kv.type == NUT_F16)
        tree_in<NUT_F16>(a, plan.queries, grid, stream);
    else
        tree_in<NUT_BF16>(a, plan.queries, grid, stream);
    check_launch("tree attention");
    if (plan.runs == 1)
        return;
    const uint64_t threads = uint64_t(draft.most) * heads * (kv.head_dim / 4);
    hipLaunchKernelGGL(tree_join_kernel, dim3(uint32_t((threads + 255) / 256), draft.batch),
                       dim3(256), 0, stream, a);
    check_launch("tree attention");
}

} // namespace nut
