// The paged KV cache's index arithmetic (nutllm_amd/csrc/paged_index.hpp) as
// the kernels use it, on the host: every row lands in its page and slot, an
// append's workgroups cover its rows once, and pages, lengths and counts that
// a call cannot follow are refused before anything is read or written.
#include <algorithm>
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "paged_index.hpp"

using namespace nut;

static void expect(bool ok, const char *what, long a = 0, long b = 0, long c = 0)
{
    if (!ok) {
        std::printf("FAILED: %s (%ld, %ld, %ld)\n", what, a, b, c);
        std::exit(1);
    }
}

static void division()
{
    std::mt19937_64 rng(1);
    for (int t = 0; t < 60000; t++) {
        const uint32_t size =
            t < 5000 ? uint32_t(t + 1) : uint32_t(1 + (rng() % 0x7fffffffu >> (rng() % 31)));
        const PageDivision d = page_division(size);
        for (int k = 0; k < 40; k++) {
            const int64_t row = int64_t((rng() & 0x7fffffffu) >> (rng() % 31));
            const int64_t edge = row / size * size;
            for (int64_t x : {row, edge, edge - 1, edge + size - 1, int64_t(0x7fffffff)})
                if (x >= 0 && x <= 0x7fffffff)
                    expect(divide(d, uint32_t(x)) == uint32_t(x) / size, "division", size, x);
        }
    }
}

static void spans()
{
    std::mt19937 rng(2);
    for (int t = 0; t < 20000; t++) {
        const uint32_t size = 1 + rng() % 70, n = rng() % 300, max_new = 1 + rng() % 200;
        const uint32_t m = 1 + rng() % max_new;
        const PageDivision d = page_division(size);
        std::vector<int> seen(n + m + size, 0);
        const uint32_t touched = pages_touched(max_new, size);
        for (uint32_t c = 0; c < touched; c++) {
            const AppendSpan s = append_span(n, m, c, size, d);
            for (uint32_t r = s.begin; r < s.end; r++) {
                expect(r / size == s.index, "row in its page", n, m, r);
                seen[r]++;
            }
        }
        for (uint32_t r = 0; r < seen.size(); r++)
            expect(seen[r] == (r >= n && r < n + m), "each row once", n, m, r);
    }
    // the last page of the longest sequence
    const PageDivision d = page_division(48);
    const uint32_t n = 0x7fffffffu - 4096 - 5;
    const AppendSpan s = append_span(n, 5, 0, 48, d);
    expect(s.begin == n && s.end > s.begin && s.end <= n + 5, "long sequence", s.begin, s.end);
    expect(append_span(n, 5, 3, 48, d).begin == append_span(n, 5, 3, 48, d).end, "behind it");
}

static void threads()
{
    for (uint32_t dim = 8; dim <= 256; dim += 8)
        for (uint32_t size : {1u, 3u, 16u, 1u << 26, 1u << 27, 1u << 28, 0x7fffffffu})
            for (uint32_t max_new : {1u, 2u, 64u, 1u << 27, 1u << 28, 1u << 29, 0x7fffffffu}) {
                const uint32_t t = append_threads(size, max_new, dim);
                const uint64_t rows = std::min(size, max_new), all = rows * (dim / 8);
                expect(t % 64 == 0 && t <= 256 && t >= dim / 8, "append threads", dim, size, t);
                expect(t == 256 || (t >= all && t < all + 64), "a page's rows", dim, size, t);
            }
}

static void refusals()
{
    for (int page : {0, 1, 9})
        expect(page_in(page, 10), "page", page);
    for (int page : {-1, INT_MIN, 10, 11, INT_MAX})
        expect(!page_in(page, 10), "bad page", page);
    for (int n : {0, 1, 32})
        expect(length_in(n, 32), "length", n);
    for (int n : {-1, INT_MIN, 33, INT_MAX})
        expect(!length_in(n, 32), "bad length", n);
    expect(append_error(20, 0, 12, 12, 40, 32) == 0, "fits");
    expect(append_error(20, 28, 12, 12, 40, 32) == 0, "the last source rows");
    expect(append_error(0, 5, 0, 12, 40, 32) == 0, "no rows");
    expect(append_error(20, 0, 13, 13, 40, 32) == kBadLength, "past max_length");
    expect(append_error(-1, 0, 1, 12, 40, 32) == kBadLength, "negative length");
    expect(append_error(INT_MAX, 0, 12, 12, 40, 32) == kBadLength, "length at the type's end");
    expect(append_error(20, 0, 13, 12, 40, 32) == kBadRows, "over max_new");
    expect(append_error(20, 29, 12, 12, 40, 32) == kBadRows, "past the source");
    expect(append_error(20, -1, 2, 12, 40, 32) == kBadRows, "before the source");
    expect(append_error(20, 5, -1, 12, 40, 32) == kBadRows, "starts that fall");
    expect(append_error(0, INT_MAX, int64_t(INT_MIN) - INT_MAX, 12, 40, 32) == kBadRows,
           "the widest fall");
}

int main()
{
    division();
    spans();
    threads();
    refusals();
    std::printf("all passed\n");
    return 0;
}
