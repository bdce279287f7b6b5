// capi_paged.cpp — the extern "C" entry points of the paged KV cache
// declared in include/nutllm_hip.h: every argument that the host can see is
// checked here, before anything is launched.
#include <algorithm>
#include <cmath>

#include "model.hpp"
#include "paged_checks.hpp"

namespace {

using namespace nut::checks;
using nut::require;

nut::PagedHistory history_of(const nut::PagedSeqs &s, const nut_paged_history *h)
{
    if (h == nullptr)
        return nut::PagedHistory{nullptr, nullptr, 0};
    require(h->d_weights != nullptr && h->d_positions != nullptr, NUT_EINVAL,
            "paged cache: null history");
    require(h->stride >= s.max_length && h->stride <= kMost, NUT_EINVAL,
            "paged cache: history shorter than the longest sequence");
    return nut::PagedHistory{h->d_weights, h->d_positions, h->stride};
}

uint32_t top_of(const nut::PagedView &kv, size_t top)
{
    require(top != 0 && top <= kMost && double(top) * double(kv.page_size) <= double(kMost - 4096),
            NUT_EINVAL, "paged cache: invalid selection");
    return uint32_t(top);
}

// `each` rows a sequence where starts is null.
void append(const nut_paged_kv *kv, const nut_paged_batch *seqs, const float *keys,
            const float *values, size_t rows, size_t row_stride, size_t head_stride,
            const int *starts, size_t each, size_t max_new, const nut_paged_history *history,
            const int *firsts, int *new_lengths, void *stream)
{
    const nut::PagedView v = view_of(kv);
    const nut::PagedSeqs s = seqs_of(v, seqs);
    const nut::PagedHistory h = history_of(s, history);
    require(keys != nullptr && values != nullptr, NUT_EINVAL, "paged cache: null pointer");
    require(apart(new_lengths, s.lengths, s.batch, s.batch), NUT_EINVAL,
            "paged cache: new lengths must not be the lengths");
    require(max_new != 0 && max_new <= kMost && rows <= kMost, NUT_EINVAL,
            "paged append: invalid row count");
    require(starts != nullptr || (max_new == std::max(each, size_t(1)) &&
                                  rows / std::max(each, size_t(1)) >= s.batch) || each == 0,
            NUT_EINVAL, "paged append: one row a sequence without starts");
    if (head_stride == 0)
        head_stride = v.head_dim;
    if (row_stride == 0)
        row_stride = size_t(v.kv_heads) * v.head_dim;
    require(aligned16(keys) && aligned16(values) && row_stride % 4 == 0 && head_stride % 4 == 0,
            NUT_EINVAL, "paged cache: rows must start at multiples of 16 bytes");
    require(row_stride < (size_t(1) << 31) && head_stride < (size_t(1) << 31), NUT_EINVAL,
            "paged append: invalid strides");
    extent(v.head_dim, {Axis{row_stride, rows}, Axis{head_stride, v.kv_heads}});
    require(apart(new_lengths, starts, s.batch, size_t(s.batch) + 1) &&
                apart(new_lengths, firsts, s.batch, s.batch),
            NUT_EINVAL, "paged append: new lengths must not be the starts or first positions");
    nut::ensure_device();
    // a sequence that gained more than max_length rows would be refused
    nut::launch_paged_append(v, s, keys, values, rows, row_stride, head_stride, starts,
                             uint32_t(each), uint32_t(std::min(max_new, size_t(s.max_length))),
                             h, firsts, new_lengths, as_stream(stream));
}

} // namespace

extern "C" {

int nut_paged_append(const nut_paged_kv *kv, const nut_paged_batch *seqs, const float *d_keys,
                     const float *d_values, size_t rows, size_t row_stride, size_t head_stride,
                     const int *d_starts, size_t max_new, const nut_paged_history *history,
                     const int *d_first_positions, int *d_new_lengths, void *stream)
{
    return nut::guarded([&]() {
        append(kv, seqs, d_keys, d_values, rows, row_stride, head_stride, d_starts, 1, max_new,
               history, d_first_positions, d_new_lengths, stream);
    });
}

size_t nut_paged_attention_workspace(const nut_paged_kv *kv, const nut_paged_batch *seqs,
                                     size_t heads, size_t top, int weighted)
{
    return bytes_or_error([&]() {
        const nut::PagedView v = view_of(kv);
        const nut::PagedSeqs s = seqs_of(v, seqs);
        require(top == 0 || weighted == 0, NUT_EINVAL,
                "paged attention: no weights of a selection");
        return nut::plan_attention(v, s, heads_of(v, heads), top == 0 ? 0 : top_of(v, top),
                                   weighted != 0)
            .bytes;
    });
}

int nut_paged_attention(const nut_paged_kv *kv, const nut_paged_batch *seqs,
                        const float *d_query, size_t query_stride, size_t heads, float scale,
                        const int *d_selected, size_t top, const nut_paged_history *history,
                        float *d_out, float *d_lse, void *d_workspace, size_t workspace_bytes,
                        void *stream)
{
    return nut::guarded([&]() {
        const nut::PagedView v = view_of(kv);
        const nut::PagedSeqs s = seqs_of(v, seqs);
        const uint32_t n = heads_of(v, heads);
        query_stride = query_stride_of(v, d_query, query_stride, n);
        require(std::isfinite(scale), NUT_EINVAL, "paged attention: scale is not finite");
        require((d_selected == nullptr) == (top == 0), NUT_EINVAL,
                "paged cache: invalid selection");
        require(d_selected == nullptr || history == nullptr, NUT_EINVAL,
                "paged attention: no weights of a selection");
        const uint32_t chosen = top == 0 ? 0 : top_of(v, top);
        const nut::PagedHistory h = history_of(s, history);
        require(d_out != nullptr, NUT_EINVAL, "paged cache: null pointer");
        require(aligned16(d_out), NUT_EINVAL,
                "paged cache: rows must start at multiples of 16 bytes");
        check_workspace(d_workspace, workspace_bytes,
                        nut::plan_attention(v, s, n, chosen, history != nullptr).bytes);
        nut::ensure_device();
        nut::launch_paged_attention(v, s, d_query, query_stride, n, scale, d_selected, chosen, h,
                                    d_out, d_lse, static_cast<char *>(d_workspace),
                                    as_stream(stream));
    });
}

size_t nut_paged_select_workspace(const nut_paged_kv *kv, const nut_paged_batch *seqs,
                                  size_t heads, size_t top)
{
    return bytes_or_error([&]() {
        const nut::PagedView v = view_of(kv);
        const nut::PagedSeqs s = seqs_of(v, seqs);
        (void)heads_of(v, heads), (void)top_of(v, top);
        return nut::select_workspace(v, s);
    });
}

int nut_paged_select(const nut_paged_kv *kv, const nut_paged_batch *seqs, const float *d_query,
                     size_t query_stride, size_t heads, size_t top, size_t first, size_t last,
                     int *d_selected, void *d_workspace, size_t workspace_bytes, void *stream)
{
    return nut::guarded([&]() {
        const nut::PagedView v = view_of(kv);
        const nut::PagedSeqs s = seqs_of(v, seqs);
        const uint32_t n = heads_of(v, heads);
        query_stride = query_stride_of(v, d_query, query_stride, n);
        require(v.bounds != nullptr, NUT_EINVAL, "paged select: the cache keeps no bounds");
        const uint32_t chosen = top_of(v, top);
        require(first <= top && last <= top - first, NUT_EINVAL,
                "paged select: first and last pages exceed the selection");
        require(d_selected != nullptr, NUT_EINVAL, "paged cache: null pointer");
        check_workspace(d_workspace, workspace_bytes, nut::select_workspace(v, s));
        nut::ensure_device();
        nut::launch_paged_select(v, s, d_query, query_stride, n, chosen, uint32_t(first),
                                 uint32_t(last), d_selected, static_cast<char *>(d_workspace),
                                 as_stream(stream));
    });
}

size_t nut_paged_evict_workspace(const nut_paged_kv *kv, const nut_paged_batch *seqs,
                                 size_t budget)
{
    return bytes_or_error([&]() {
        const nut::PagedView v = view_of(kv);
        const nut::PagedSeqs s = seqs_of(v, seqs);
        require(budget != 0 && budget <= kMost, NUT_EINVAL, "paged evict: invalid budget");
        return nut::evict_workspace(v, s, uint32_t(budget));
    });
}

int nut_paged_evict(const nut_paged_kv *kv, const nut_paged_batch *seqs,
                    const nut_paged_history *history, size_t budget, size_t first, size_t last,
                    int *d_new_lengths, void *d_workspace, size_t workspace_bytes, void *stream)
{
    return nut::guarded([&]() {
        const nut::PagedView v = view_of(kv);
        const nut::PagedSeqs s = seqs_of(v, seqs);
        require(history != nullptr, NUT_EINVAL, "paged cache: null history");
        const nut::PagedHistory h = history_of(s, history);
        require(budget != 0 && budget <= kMost, NUT_EINVAL, "paged evict: invalid budget");
        require(first <= budget && last <= budget - first, NUT_EINVAL,
                "paged evict: first and last rows exceed the budget");
        require(d_new_lengths != nullptr, NUT_EINVAL, "paged cache: null pointer");
        require(apart(d_new_lengths, s.lengths, s.batch, s.batch), NUT_EINVAL,
                "paged cache: new lengths must not be the lengths");
        check_workspace(d_workspace, workspace_bytes,
                        nut::evict_workspace(v, s, uint32_t(budget)));
        nut::ensure_device();
        nut::launch_paged_evict(v, s, h, uint32_t(budget), uint32_t(first), uint32_t(last),
                                d_new_lengths, static_cast<char *>(d_workspace),
                                as_stream(stream));
    });
}

int nut_paged_append_cache(const nut_paged_kv *kv, const nut_paged_batch *seqs,
                           const nut_kvcache *source, size_t layer, size_t begin, size_t end,
                           const nut_paged_history *history, const int *d_first_positions,
                           int *d_new_lengths, void *stream)
{
    return nut::guarded([&]() {
        require(source != nullptr, NUT_EINVAL, "kv cache: null cache");
        const nut::PagedView v = view_of(kv);
        const nut_config &c = source->config;
        require(source->kv_heads() == v.kv_heads && c.head_dim == v.head_dim, NUT_EINVAL,
                "paged append: cache configuration mismatch");
        require(layer < c.layers && begin <= end && end <= source->length, NUT_EOUTOFRANGE,
                "kv cache: index out of range");
        require(seqs != nullptr && seqs->batch == 1, NUT_EINVAL, "paged cache: invalid batch");
        const size_t row = c.head_dim, head = c.max_seq * row;
        const size_t at = layer * source->layer_elements() + begin * row, rows = end - begin;
        append(kv, seqs, source->keys.as<float>() + at, source->values.as<float>() + at, rows, row,
               head, nullptr, rows, std::max(rows, size_t(1)), history, d_first_positions,
               d_new_lengths, stream);
    });
}

int nut_status_check(int *d_status)
{
    return nut::guarded([&]() {
        require(d_status != nullptr, NUT_EINVAL, "paged cache: no status word");
        nut::ensure_device();
        nut::hip_check(hipDeviceSynchronize(), "hipDeviceSynchronize");
        int bits = 0;
        nut::hip_check(hipMemcpy(&bits, d_status, sizeof bits, hipMemcpyDeviceToHost),
                       "hipMemcpy to host");
        if (bits == 0)
            return;
        const int zero = 0;
        nut::hip_check(hipMemcpy(d_status, &zero, sizeof zero, hipMemcpyHostToDevice),
                       "hipMemcpy to device");
        require((bits & nut::kBadPage) == 0, NUT_EOUTOFRANGE, "paged cache: page out of range");
        require((bits & nut::kBadLength) == 0, NUT_EOUTOFRANGE,
                "paged cache: length out of range");
        require((bits & nut::kBadRows) == 0, NUT_EOUTOFRANGE, "paged cache: rows out of range");
        require((bits & nut::kBadTree) == 0, NUT_EOUTOFRANGE, "draft tree: parent out of range");
        require((bits & nut::kBadParent) == 0, NUT_EOUTOFRANGE, "page pool: parent out of range");
        nut::fail(NUT_EOUTOFRANGE, "page pool: out of pages");
    });
}

int nut_paged_check(const nut_paged_kv *kv)
{
    return nut_status_check(kv == nullptr ? nullptr : kv->d_status);
}

} // extern "C"
