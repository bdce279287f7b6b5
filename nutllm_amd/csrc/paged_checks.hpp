// paged_checks.hpp — what the entry points over a paged KV cache check of their
// arguments before anything is launched (capi_paged.cpp, capi_serving.cpp).
#pragma once

#include <algorithm>

#include "paged.hpp"
#include "runtime.hpp"

namespace nut::checks {

constexpr size_t kMost = 0x7fffffff;

inline hipStream_t as_stream(void *stream) { return static_cast<hipStream_t>(stream); }

inline bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

struct Axis {
    size_t stride, count;
};

// Elements that rows of head_dim span along these axes. The strides, widest
// first, each have to clear what lies inside them.
template <size_t N> double extent(size_t head_dim, const Axis (&axes)[N])
{
    Axis axis[N];
    std::copy(axes, axes + N, axis);
    std::sort(axis, axis + N, [](const Axis &a, const Axis &b) {
        return a.stride != b.stride ? a.stride < b.stride : a.count < b.count;
    });
    double inside = double(head_dim);
    for (const Axis &a : axis) {
        if (a.count <= 1)
            continue;
        require(double(a.stride) >= inside, NUT_EINVAL, "paged cache: rows overlap");
        inside += double(a.stride) * double(a.count - 1);
    }
    return inside;
}

inline PagedView view_of(const nut_paged_kv *kv)
{
    require(kv != nullptr && kv->d_keys != nullptr && kv->d_values != nullptr, NUT_EINVAL,
            "paged cache: null pointer");
    require(kv->type == NUT_F32 || kv->type == NUT_F16 || kv->type == NUT_BF16, NUT_EINVAL,
            "paged cache: unknown type");
    require(kv->pages != 0 && kv->pages <= kMost && kv->page_size != 0 &&
                kv->page_size <= kMost && kv->kv_heads != 0 && kv->kv_heads <= kMost,
            NUT_EINVAL, "paged cache: invalid dimensions");
    require(kv->head_dim != 0 && kv->head_dim % 8 == 0 && kv->head_dim <= 256, NUT_EINVAL,
            "paged cache: head dim must be a multiple of 8 up to 256");
    const size_t size = paged_element(kv->type);
    PagedView v{};
    v.keys = static_cast<char *>(kv->d_keys);
    v.values = static_cast<char *>(kv->d_values);
    v.bounds = static_cast<char *>(kv->d_bounds);
    v.pages = uint32_t(kv->pages), v.page_size = uint32_t(kv->page_size);
    v.kv_heads = uint32_t(kv->kv_heads), v.head_dim = uint32_t(kv->head_dim);
    v.type = kv->type, v.status = kv->d_status;
    v.division = page_division(v.page_size);
    // Rows are at most 2^93 elements apart by these counts; offsets have to
    // stay below 2^63 bytes.
    const double rows = double(kv->pages) * double(kv->page_size) * double(kv->kv_heads);
    require(rows * double(kv->head_dim) * double(size) < 9e18, NUT_EINVAL,
            "paged cache: invalid dimensions");
    if (kv->page_stride == 0 && kv->head_stride == 0 && kv->slot_stride == 0) {
        v.slot_stride = kv->head_dim * size;
        v.head_stride = kv->page_size * v.slot_stride;
        v.page_stride = kv->kv_heads * v.head_stride;
    } else {
        const double inside = extent(kv->head_dim, {Axis{kv->page_stride, kv->pages},
                                                    Axis{kv->head_stride, kv->kv_heads},
                                                    Axis{kv->slot_stride, kv->page_size}});
        require(inside * double(size) < 9e18 && kv->page_stride < (size_t(1) << 60) &&
                    kv->head_stride < (size_t(1) << 60) && kv->slot_stride < (size_t(1) << 60),
                NUT_EINVAL, "paged cache: invalid dimensions");
        v.page_stride = kv->page_stride * size;
        v.head_stride = kv->head_stride * size;
        v.slot_stride = kv->slot_stride * size;
    }
    require(aligned16(kv->d_keys) && aligned16(kv->d_values) && aligned16(kv->d_bounds) &&
                v.page_stride % 16 == 0 && v.head_stride % 16 == 0 && v.slot_stride % 16 == 0,
            NUT_EINVAL, "paged cache: rows must start at multiples of 16 bytes");
    return v;
}

inline PagedSeqs seqs_of(const PagedView &kv, const nut_paged_batch *s)
{
    require(s != nullptr && s->d_pages != nullptr && s->d_lengths != nullptr, NUT_EINVAL,
            "paged cache: null pointer");
    require(s->batch != 0 && s->batch <= kMost && s->max_length != 0 &&
                s->max_length <= kMost - 4096 && s->table_stride <= kMost,
            NUT_EINVAL, "paged cache: invalid batch");
    require(double(s->table_stride) * double(kv.page_size) >= double(s->max_length), NUT_EINVAL,
            "paged cache: page table shorter than the longest sequence");
    return PagedSeqs{s->d_pages, s->d_lengths, uint32_t(s->table_stride),
                          uint32_t(s->batch), uint32_t(s->max_length)};
}

inline uint32_t heads_of(const PagedView &kv, size_t heads)
{
    require(heads != 0 && heads <= kMost && heads % kv.kv_heads == 0, NUT_EINVAL,
            "paged cache: heads must be a multiple of the KV heads");
    return uint32_t(heads);
}

inline size_t query_stride_of(const PagedView &kv, const float *query, size_t stride, size_t heads)
{
    require(query != nullptr, NUT_EINVAL, "paged cache: null pointer");
    if (stride == 0)
        stride = heads * kv.head_dim;
    require(aligned16(query) && stride % 4 == 0, NUT_EINVAL,
            "paged cache: rows must start at multiples of 16 bytes");
    require(stride >= heads * kv.head_dim, NUT_EINVAL, "paged cache: rows overlap");
    return stride;
}

inline void check_workspace(const void *workspace, size_t bytes, size_t need)
{
    require(need == 0 || (workspace != nullptr && bytes >= need), NUT_EINVAL,
            "paged cache: workspace too small");
    require(aligned16(workspace), NUT_EINVAL, "paged cache: workspace must be 16-byte aligned");
}

// New lengths are written while other workgroups still read a call's inputs.
inline bool apart(const int *written, const int *read, size_t batch, size_t count)
{
    const uintptr_t a = reinterpret_cast<uintptr_t>(written), b = reinterpret_cast<uintptr_t>(read);
    return written == nullptr || read == nullptr || a + batch * sizeof(int) <= b ||
           b + count * sizeof(int) <= a;
}

// The bytes that `body` finds, or (size_t)-1 where it refuses its arguments.
template <typename Body> size_t bytes_or_error(Body &&body)
{
    size_t bytes = 0;
    return guarded([&]() { bytes = body(); }) == NUT_OK ? bytes : size_t(-1);
}

} // namespace nut::checks
