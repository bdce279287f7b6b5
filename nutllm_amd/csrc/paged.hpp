// paged.hpp — views and launches of the paged KV cache kernels
// (paged_attention.hip, paged_cache.hip), called from capi_paged.cpp after
// the host has checked every argument.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "nutllm_hip.h"
#include "status.hpp"

namespace nut {

// Bits of a view's status word.
enum : int { kBadPage = 1, kBadLength = 2, kBadRows = 4 };

// A nut_paged_kv with its strides resolved, in bytes.
struct PagedView {
    char *keys, *values, *bounds;
    uint32_t pages, page_size, kv_heads, head_dim;
    uint32_t page_magic, page_shift; // row / page_size, see page_of
    size_t page_stride, head_stride, slot_stride;
    int type;
    int *status;
};

// Division of rows (below 2^31) by the page size as a multiplication: with
// 2^(l - 1) < size <= 2^l and magic = floor(2^(31 + l) / size) + 1, the product
// row magic exceeds row 2^(31 + l) / size by at most row < 2^31, less than
// what a row's fraction of a page is short of the next one. Size 1: magic 0.
inline void set_page_division(PagedView &v)
{
    uint32_t l = 0;
    while ((uint64_t(1) << l) < v.page_size)
        l++;
    v.page_magic = l == 0 ? 0 : uint32_t((uint64_t(1) << (31 + l)) / v.page_size + 1);
    v.page_shift = l == 0 ? 0 : l - 1;
}

inline __host__ __device__ uint32_t page_of(const PagedView &v, uint32_t row)
{
    return v.page_magic == 0 ? row
                             : uint32_t(uint64_t(row) * v.page_magic >> 32) >> v.page_shift;
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
    require(workgroups * threads <= 0xffffffffull, NUT_EINVAL,
            "paged cache: more rows than one launch covers");
    return dim3(uint32_t(workgroups));
}

inline size_t paged_element(int type) { return type == NUT_F32 ? 4 : 2; }

// How an attention call is split: `chunks` runs of `chunk` rows (of the
// sequence, or of the selection) a sequence and KV head, `tiles` tiles of 16
// query heads, and where the pieces of its workspace lie.
struct AttentionPlan {
    uint32_t chunk, chunks, tiles;
    size_t parts, stats, scores; // byte offsets
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
