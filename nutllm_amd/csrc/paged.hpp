// paged.hpp — views and launches of the paged KV cache kernels
// (paged_attention.hip, paged_cache.hip), called from capi_paged.cpp after
// the host has checked every argument.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "nutllm_hip.h"
#include "paged_index.hpp"
#include "status.hpp"

namespace nut {

// A nut_paged_kv with its strides resolved, in bytes.
struct PagedView {
    char *keys, *values, *bounds;
    uint32_t pages, page_size, kv_heads, head_dim;
    PageDivision division; // by page_size
    size_t page_stride, head_stride, slot_stride;
    int type;
    int *status;
};

inline __host__ __device__ uint32_t page_of(const PagedView &v, uint32_t row)
{
    return divide(v.division, row);
}

struct PagedSeqs {
    const int *table;
    const int *lengths;
    uint32_t table_stride, batch, max_length;
};

struct PagedHistory {
    float *weights; // nullptr: none
    int *positions;
    size_t stride;
};

// A grid of `workgroups` x `threads` holds at most 2^32 - 1 threads.
inline dim3 paged_grid(uint64_t workgroups, uint32_t threads)
{
    require(workgroups <= 0xffffffffull / threads, NUT_EINVAL, // their product may pass 64 bits
            "paged cache: more rows than one launch covers");
    return dim3(uint32_t(workgroups));
}

inline size_t paged_element(int type) { return type == NUT_F32 ? 4 : 2; }

// How an attention call is split: `chunks` runs of `chunk` rows (of the
// sequence, or of the selection) a sequence and KV head, `tiles` tiles of 16
// query heads, and where the pieces of its workspace lie behind the runs'
// unnormalised results. Raises NUT_EINVAL where a launch does not cover it.
struct AttentionPlan {
    uint32_t chunk, chunks, tiles;
    uint32_t likely; // rows of the longest sequence that are read, but for pages named twice
    uint32_t join_threads, weigh_blocks; // of the second launch
    size_t stats, scores; // byte offsets
    size_t bytes;
};
AttentionPlan plan_attention(const PagedView &kv, const PagedSeqs &seqs, uint32_t heads,
                             uint32_t top, bool weighted);

void launch_paged_attention(const PagedView &kv, const PagedSeqs &seqs, const float *query,
                            size_t query_stride, uint32_t heads, float scale,
                            const int *selected, uint32_t top, const PagedHistory &history,
                            float *out, float *lse, char *workspace, hipStream_t stream);

void launch_paged_append(const PagedView &kv, const PagedSeqs &seqs, const float *keys,
                         const float *values, size_t rows, size_t row_stride,
                         size_t head_stride, const int *starts, uint32_t each,
                         uint32_t max_new, const PagedHistory &history, const int *firsts,
                         int *new_lengths, hipStream_t stream);

size_t select_workspace(const PagedView &kv, const PagedSeqs &seqs);
void launch_paged_select(const PagedView &kv, const PagedSeqs &seqs, const float *query,
                         size_t query_stride, uint32_t heads, uint32_t top, uint32_t first,
                         uint32_t last, int *selected, char *workspace, hipStream_t stream);

size_t evict_workspace(const PagedView &kv, const PagedSeqs &seqs, uint32_t budget);
void launch_paged_evict(const PagedView &kv, const PagedSeqs &seqs, const PagedHistory &history,
                        uint32_t budget, uint32_t first, uint32_t last, int *new_lengths,
                        char *workspace, hipStream_t stream);

} // namespace nut
