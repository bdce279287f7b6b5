// serving.hpp — views and launches of what serves several continuations of a
// text: draft trees (tree_attention.hip, draft.hip), page pools (pages.hip)
// and beam search (beam.hip), called from capi_serving.cpp after the host has
// checked every argument.
#pragma once

#include "paged.hpp"

namespace nut {

constexpr uint32_t kMostNodes = 1024;  // of a draft tree
constexpr uint32_t kMostLayers = 64;   // of a launch
constexpr uint32_t kMostBeams = 64;
constexpr uint32_t kMostVocab = 262144;

struct DraftView {
    const int *starts, *parents;
    uint32_t *mask;
    size_t mask_stride;
    uint32_t total, most, batch;
    int *status;
};

// Layers of one shape: `view` with each layer's pointers in the place of its own.
struct PagedLayers {
    PagedView view;
    uint32_t count;
    char *keys[kMostLayers], *values[kMostLayers], *bounds[kMostLayers];
};

struct PoolView {
    int *refs;
    uint32_t pages, page_size;
    int *status;
};

struct TableView {
    int *pages, *lengths, *held;
    uint32_t stride, batch;
};

struct BeamsView {
    float *scores;
    int *lengths, *ended;
    uint32_t requests, beams;
};

// How a tree attention call is split. Few query rows (nodes times the heads that
// share a KV head): `runs` runs of `run` rows of a sequence. Many: `shares`
// workgroups that share out blocks of 64 query rows and stages of rows.
struct TreePlan {
    bool staged, past; // past the caches
    uint32_t waves; // of a workgroup that hold different query rows
    uint32_t blocks, run, runs, shares;
    uint32_t teams; // of the join; 0: none
    size_t stats, before; // byte offsets of the parts' sums, of the stages before each sequence
    size_t bytes;
};
TreePlan plan_tree(const PagedView &kv, const PagedSeqs &seqs, const DraftView &draft,
                   uint32_t heads);
void launch_tree_attention(const PagedView &kv, const PagedSeqs &seqs, const DraftView &draft,
                           const float *query, size_t query_stride, uint32_t heads, float scale,
                           float *out, float *lse, char *workspace, hipStream_t stream);

void launch_draft_mask(const DraftView &draft, int *depths, hipStream_t stream);
void launch_draft_accept(const DraftView &draft, const PagedSeqs &seqs, const int *tokens,
                         const int *chosen, int *path, size_t path_stride, int *counts, int *last,
                         int *new_lengths, hipStream_t stream);
void launch_paged_keep(const PagedLayers &layers, const PagedSeqs &seqs, const int *path,
                       size_t path_stride, const int *counts, hipStream_t stream);

size_t reorder_workspace(const PoolView &pool, const TableView &from, const TableView &to);
void launch_reorder(const PoolView &pool, const TableView &from, const TableView &to,
                    const int *parents, const int *gains, uint32_t gain, int *copies,
                    char *workspace, hipStream_t stream);
size_t compact_workspace(const PoolView &pool, const TableView &table);
void launch_compact(const PoolView &pool, const TableView &table, uint32_t limit, int *copies,
                    uint32_t count, char *workspace, hipStream_t stream);
void launch_paged_copy(const PagedLayers &layers, const int *copies, uint32_t count,
                       hipStream_t stream);

size_t beam_workspace(const BeamsView &from, const BeamsView &to, uint32_t vocab);
void launch_beam_select(const BeamsView &from, const BeamsView &to, const void *logits, int type,
                        size_t row_stride, uint32_t vocab, int eos, float power, int *parents,
                        int *tokens, char *workspace, hipStream_t stream);
void launch_beam_gather(const char *source, size_t from_stride, uint32_t sources, char *to,
                        size_t to_stride, uint32_t rows, size_t row_bytes, const int *parents,
                        int *status, hipStream_t stream);

#ifdef __HIPCC__
__device__ __forceinline__ void status_flag(int *status, int bit)
{
    if (status != nullptr)
        atomicOr(status, bit);
}

// Node rows [from, from + count) of sequence b; none, reported by the caller's
// `report` thread, where the starts are not ones that the draft allows.
struct NodeSpan {
    uint32_t from, count;
};
__device__ __forceinline__ NodeSpan nodes_of(const DraftView &d, uint32_t b, bool report)
{
    if (d.starts == nullptr)
        return NodeSpan{b * d.most, d.most};
    const int from = d.starts[b], end = d.starts[b + 1];
    if (span_in(from, end, d.most, d.total))
        return NodeSpan{uint32_t(from), uint32_t(end - from)};
    if (report)
        status_flag(d.status, kBadRows);
    return NodeSpan{0, 0};
}
#endif

} // namespace nut
