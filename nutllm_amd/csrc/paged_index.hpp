// paged_index.hpp — where rows of a paged KV cache lie, and which pages,
// lengths and row counts a call can follow. Plain integer arithmetic, the same
// on the host and in kernels.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define NUT_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define NUT_HOST_DEVICE inline
#endif

namespace nut {

// Bits of a view's status word.
enum : int { kBadPage = 1, kBadLength = 2, kBadRows = 4 };

// Division of rows (below 2^31) by the page size as a multiplication: with
// 2^(l - 1) < size <= 2^l and magic = floor(2^(31 + l) / size) + 1, the product
// row magic exceeds row 2^(31 + l) / size by at most row < 2^31, less than
// what a row's fraction of a page is short of the next one. Size 1: magic 0.
struct PageDivision {
    uint32_t magic, shift;
};

inline PageDivision page_division(uint32_t size)
{
    uint32_t l = 0;
    while ((uint64_t(1) << l) < size)
        l++;
    if (l == 0)
        return PageDivision{0, 0};
    return PageDivision{uint32_t((uint64_t(1) << (31 + l)) / size + 1), l - 1};
}

NUT_HOST_DEVICE uint32_t divide(PageDivision d, uint32_t row)
{
    return d.magic == 0 ? row : uint32_t(uint64_t(row) * d.magic >> 32) >> d.shift;
}

// A page that the cache has.
NUT_HOST_DEVICE bool page_in(int page, uint32_t pages)
{
    return page >= 0 && uint32_t(page) < pages;
}

// A length that a call allows.
NUT_HOST_DEVICE bool length_in(int length, uint32_t most)
{
    return length >= 0 && uint32_t(length) <= most;
}

// 0, or why `gain` source rows from `from` on, of `rows`, cannot go behind
// `length` rows.
NUT_HOST_DEVICE int append_error(int length, int64_t from, int64_t gain, uint32_t max_new,
                                 uint64_t rows, uint32_t max_length)
{
    if (from < 0 || gain < 0 || gain > int64_t(max_new) || from + gain > int64_t(rows))
        return kBadRows;
    if (length < 0 || length + gain > int64_t(max_length))
        return kBadLength;
    return 0;
}

// Pages that `gain` rows (one or more) can lie in, wherever they begin.
NUT_HOST_DEVICE uint32_t pages_touched(uint32_t gain, uint32_t page_size)
{
    return (gain - 1 + page_size - 1) / page_size + 1;
}

// Threads of an append's workgroup: head_dim / 8 a row, as many rows as a page
// gains at most, in whole waves up to 256 (and never fewer than one row's).
NUT_HOST_DEVICE uint32_t append_threads(uint32_t page_size, uint32_t max_new, uint32_t head_dim)
{
    const uint32_t rows = page_size < max_new ? page_size : max_new;
    const uint64_t threads = (uint64_t(rows) * (head_dim / 8) + 63) / 64 * 64;
    return threads < 256 ? uint32_t(threads) : 256;
}

// The rows [begin, end) that an append of m rows behind n puts into the c-th
// page it touches, page `index` of the sequence; begin = end for none.
struct AppendSpan {
    uint32_t index, begin, end;
};

NUT_HOST_DEVICE AppendSpan append_span(uint32_t n, uint32_t m, uint32_t c, uint32_t page_size,
                                       PageDivision d)
{
    const uint32_t index = divide(d, n) + c;
    const uint64_t first = uint64_t(index) * page_size, behind = uint64_t(n) + m;
    if (first >= behind)
        return AppendSpan{index, 0, 0};
    const uint64_t end = first + page_size < behind ? first + page_size : behind;
    return AppendSpan{index, first > n ? uint32_t(first) : n, uint32_t(end)};
}

} // namespace nut
