// draft.hip — a draft tree beside its attention: the nodes' masks, the path that
// the model agrees with, and the cache rows that stay.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "device.hpp"
#include "paged_device.hpp"
#include "runtime.hpp"
#include "serving.hpp"

namespace nut {

namespace {

// The parent of node i, a number below i, or -1; others are reported.
__device__ __forceinline__ int parent_of(const DraftView &d, uint32_t from, uint32_t i)
{
    const int parent = d.parents[from + i];
    if (parent_in(parent, i))
        return parent;
    status_flag(d.status, kBadTree);
    return -1;
}

// A workgroup a sequence, a thread a node: it goes up the tree, which names the
// mask's words from the last to the first, so that each is finished in a
// register. Latency bounds it: 16 trees of 64 nodes 3.0 us (2.0 at least), a launch.
__global__ void mask_kernel(DraftView d, int *depths)
{
    __shared__ int16_t parents[kMostNodes];
    const uint32_t b = blockIdx.x;
    const NodeSpan nodes = nodes_of(d, b, threadIdx.x == 0);
    for (uint32_t i = threadIdx.x; i < nodes.count; i += blockDim.x)
        parents[i] = int16_t(parent_of(d, nodes.from, i));
    __syncthreads();
    const int words = int((d.most + 31) / 32);
    for (uint32_t i = threadIdx.x; i < nodes.count; i += blockDim.x) {
        uint32_t *mask = d.mask + (nodes.from + i) * d.mask_stride;
        int depth = -1, w = words - 1;
        uint32_t bits = 0;
        for (int at = int(i); at >= 0; at = parents[at], depth++) {
            for (; w > at / 32; w--) {
                mask[w] = bits;
                bits = 0;
            }
            bits |= 1u << (at % 32);
        }
        for (; w >= 0; w--) {
            mask[w] = bits;
            bits = 0;
        }
        if (depths != nullptr)
            depths[nodes.from + i] = depth;
    }
}

// A workgroup a sequence: every node that its parent's choice names puts itself
// down as the one to go on with, the lowest staying; then one thread follows.
// Latency bounds it: 16 trees of 64 nodes 3.0 us (2.7 at least), a launch.
__global__ void accept_kernel(DraftView d, PagedSeqs s, const int *__restrict__ tokens,
                              const int *__restrict__ chosen, int *path, size_t path_stride,
                              int *counts, int *last, int *new_lengths)
{
    __shared__ int choice[kMostNodes], next[kMostNodes];
    const uint32_t b = blockIdx.x;
    const NodeSpan nodes = nodes_of(d, b, threadIdx.x == 0);
    const int length = s.lengths[b];
    for (uint32_t i = threadIdx.x; i < nodes.count; i += blockDim.x) {
        choice[i] = chosen[nodes.from + i];
        next[i] = int(kMostNodes);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < nodes.count; i += blockDim.x) {
        const int parent = parent_of(d, nodes.from, i);
        if (parent >= 0 && tokens[nodes.from + i] == choice[parent])
            atomicMin(&next[parent], int(i));
    }
    __syncthreads();
    if (threadIdx.x != 0)
        return;
    const bool fits = length_with(length, nodes.count, s.max_length);
    if (!fits)
        status_flag(d.status, kBadLength);
    int count = 0, at = 0;
    if (fits && nodes.count != 0) {
        for (int to = 0; to < int(kMostNodes); to = next[to]) {
            path[b * path_stride + count++] = to;
            at = to;
        }
        if (last != nullptr)
            last[b] = choice[at];
    }
    counts[b] = count;
    if (new_lengths != nullptr)
        new_lengths[b] = length + count;
}

// A wave per sequence, KV head and layer. head_dim / 8 lanes hold a row, eight
// components of a key and of a value each, so that the wave loads a few rows
// before it stores them; as the path ascends, no later row was stored to. A row
// stays where it is as long as the path is 0, 1, 2, .. Path, table and rows are read
// one after another, which bounds it: 16 trees, 22 layers of 4 KV heads of 64 bfloat16
// components 6.0 us (4.4 at least); 32 trees, 32 layers of 32 heads of 128 fp16 ones, four
// waves after another on a SIMD's place, 21.5 (15.5 at least; four layers a wave were
// slower).
template <int TYPE>
__global__ __launch_bounds__(kWave) void keep_kernel(PagedLayers layers, PagedSeqs s,
                                                     const int *__restrict__ path,
                                                     size_t path_stride,
                                                     const int *__restrict__ counts)
{
    constexpr uint32_t kSize = TYPE == NUT_F32 ? 4 : 2;
    const PagedView &kv = layers.view;
    const uint32_t b = blockIdx.x, h = blockIdx.y, layer = blockIdx.z;
    const bool report = threadIdx.x == 0 && h == 0 && layer == 0;
    const uint32_t tpr = kv.head_dim / 8, part = threadIdx.x % tpr, group = threadIdx.x / tpr;
    const uint32_t groups = kWave / tpr;
    const int *nodes = path + b * path_stride;
    // the first rows' places beside the length and the count, which may not reach them
    int node = group < path_stride ? nodes[group] : -1;
    int before = group != 0 && group <= path_stride ? nodes[group - 1] : -1;
    const int length = s.lengths[b], listed = counts[b];
    if (listed == 0)
        return;
    if (listed < 0 || uint64_t(listed) > path_stride || !length_in(length, s.max_length)) {
        if (report)
            status_flag(kv.status, length_in(length, s.max_length) ? kBadRows : kBadLength);
        return;
    }
    const uint32_t n = uint32_t(length), most = s.max_length - n;
    char *keys = layers.keys[layer], *values = layers.values[layer];
    __shared__ float moved[kWave][8];
    __shared__ uint32_t page_at[kWave]; // index of the page that a group's row came into; ~0: none
    for (uint32_t base = 0; base < uint32_t(listed); base += groups) {
        // the group's row, if the path is good that far
        const uint32_t k = base + group;
        const bool mine = group < groups && k < uint32_t(listed);
        if (mine && base != 0)
            node = nodes[k], before = nodes[k - 1];
        const bool bad = mine && !(node > before && uint32_t(node) < most);
        const uint64_t wrong = __ballot(bad);
        const uint32_t good = wrong == 0 ? ~0u : uint32_t(__builtin_ctzll(wrong)) / tpr;
        const bool moves = mine && group < good && uint32_t(node) != k;
        size_t from = kNoRow, to = kNoRow;
        uint32_t source = 0, index = 0;
        if (moves) {
            source = page_of(kv, n + uint32_t(node));
            index = page_of(kv, n + k);
            from = paged_row(kv, s, b, source, n + uint32_t(node) - source * kv.page_size, h);
            to = paged_row(kv, s, b, index, n + k - index * kv.page_size, h);
        }
        const bool done = moves && from != kNoRow && to != kNoRow;
        constexpr int kPieces = TYPE == NUT_F32 ? 2 : 1;
        uint4 key[kPieces] = {}, value[kPieces];
        if (done) {
#pragma unroll
            for (int i = 0; i < kPieces; i++) {
                key[i] = reinterpret_cast<const uint4 *>(keys + from + part * 8 * kSize)[i];
                value[i] = reinterpret_cast<const uint4 *>(values + from + part * 8 * kSize)[i];
            }
        }
        __syncthreads(); // every row is loaded before one is stored
        if (done) {
#pragma unroll
            for (int i = 0; i < kPieces; i++) {
                reinterpret_cast<uint4 *>(keys + to + part * 8 * kSize)[i] = key[i];
                reinterpret_cast<uint4 *>(values + to + part * 8 * kSize)[i] = value[i];
            }
        }
        if (kv.bounds != nullptr) {
            float x[8];
            load8<TYPE>(reinterpret_cast<const char *>(key), x);
#pragma unroll
            for (int i = 0; i < 8; i++)
                moved[threadIdx.x][i] = x[i];
            if (group < groups && part == 0)
                page_at[group] = done && source != index ? index : ~0u;
            __syncthreads();
            // one group widens the pages' bounds, row after row
            if (threadIdx.x < tpr)
                for (uint32_t g = 0; g < groups; g++) {
                    const uint32_t into = page_at[g];
                    if (into == ~0u)
                        continue;
                    const int page = s.table[size_t(b) * s.table_stride + into];
                    char *bounds = layers.bounds[layer] +
                                   ((size_t(page) * kv.kv_heads + h) * 2 * kv.head_dim +
                                    threadIdx.x * 8) * kSize;
                    float lo[8], hi[8];
                    load8<TYPE>(bounds, lo);
                    load8<TYPE>(bounds + kv.head_dim * kSize, hi);
                    for (; g < groups && page_at[g] == into; g++)
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float x = moved[g * tpr + threadIdx.x][i];
                            lo[i] = lower(lo[i], x), hi[i] = upper(hi[i], x);
                        }
                    g--;
                    store8<TYPE>(bounds, lo);
                    store8<TYPE>(bounds + kv.head_dim * kSize, hi);
                }
            __syncthreads();
        }
        if (wrong != 0) {
            if (report)
                status_flag(kv.status, kBadRows);
            return;
        }
    }
}

} // namespace

void launch_draft_mask(const DraftView &draft, int *depths, hipStream_t stream)
{
    const uint32_t threads = std::min((draft.most + 63) / 64 * 64, 1024u);
    hipLaunchKernelGGL(mask_kernel, paged_grid(draft.batch, threads), dim3(threads), 0, stream,
                       draft, depths);
    check_launch("draft mask");
}

void launch_draft_accept(const DraftView &draft, const PagedSeqs &seqs, const int *tokens,
                         const int *chosen, int *path, size_t path_stride, int *counts, int *last,
                         int *new_lengths, hipStream_t stream)
{
    const uint32_t threads = std::min((draft.most + 63) / 64 * 64, 1024u);
    hipLaunchKernelGGL(accept_kernel, paged_grid(draft.batch, threads), dim3(threads), 0, stream,
                       draft, seqs, tokens, chosen, path, path_stride, counts, last, new_lengths);
    check_launch("draft accept");
}

void launch_paged_keep(const PagedLayers &layers, const PagedSeqs &seqs, const int *path,
                       size_t path_stride, const int *counts, hipStream_t stream)
{
    const auto run = layers.view.type == NUT_F32   ? keep_kernel<NUT_F32>
                     : layers.view.type == NUT_F16 ? keep_kernel<NUT_F16>
                                                   : keep_kernel<NUT_BF16>;
    paged_grid(uint64_t(seqs.batch) * layers.view.kv_heads * layers.count, kWave);
    hipLaunchKernelGGL(run, dim3(seqs.batch, layers.view.kv_heads, layers.count), dim3(kWave), 0,
                       stream, layers, seqs, path, path_stride, counts);
    check_launch("paged keep");
}

} // namespace nut
