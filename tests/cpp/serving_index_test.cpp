// serving_index_test.cpp — the index arithmetic of draft trees and page pools
// (nutllm_amd/csrc/paged_index.hpp) against plain loops.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "paged_index.hpp"

using namespace nut;

static void expect(bool ok, const char *what, long long a = 0, long long b = 0)
{
    if (!ok) {
        std::printf("FAIL %s (%lld, %lld)\n", what, a, b);
        std::exit(1);
    }
}

static void masks()
{
    std::vector<uint32_t> words(5);
    for (size_t i = 0; i < words.size(); i++)
        words[i] = uint32_t(0x9e3779b9u * (i + 1)) ^ 0x5bd1e995u;
    for (uint32_t count = 0; count <= words.size(); count++)
        for (int64_t at = -70; at < 230; at++) {
            uint32_t want = 0;
            for (int k = 0; k < 32; k++) {
                const int64_t bit = at + k;
                const bool set = bit < 0 || (bit < 32 * int64_t(count) &&
                                             (words[bit / 32] >> (bit % 32) & 1));
                want |= set ? 1u << k : 0;
            }
            const uint32_t got = mask_bits(at, count, [&](uint32_t w) {
                expect(w < count, "a word that there is", w, count);
                return words[w];
            });
            expect(got == want, "mask bits", at, count);
        }
    expect(mask_bits(INT64_MIN, 0, [](uint32_t) { return 0u; }) == ~0u, "rows far before");
    expect(mask_bits(int64_t(1) << 31, 5, [](uint32_t) { return ~0u; }) == 0, "rows far behind");
}

static void spans()
{
    expect(span_in(0, 0, 4, 0) && span_in(3, 7, 4, 7) && span_in(7, 7, 4, 7), "spans");
    expect(!span_in(-1, 3, 4, 7) && !span_in(3, 2, 4, 7) && !span_in(3, 8, 5, 7), "outside");
    expect(!span_in(2, 7, 4, 7), "over the most");
    expect(!span_in(INT_MIN, INT_MAX, 1024, INT_MAX), "the widest");
    expect(!span_in(INT_MAX, INT_MIN, 1024, INT_MAX), "the widest fall");
    for (int n : {0, 1, 31, 32})
        expect(length_with(n, 32 - n, 32) && !length_with(n, 33 - n, 32), "lengths", n);
    expect(!length_with(-1, 0, 32) && !length_with(INT_MIN, 5, UINT32_MAX), "negative lengths");
    expect(!length_with(INT_MAX, 1024, INT_MAX), "length at the type's end");
    for (int i : {0, 1, 5, 1023}) {
        expect(parent_in(-1, i) && !parent_in(i, i) && !parent_in(-2, i), "parents", i);
        expect(parent_in(0, i) == (i > 0) && parent_in(i - 1, i), "the one before", i);
        expect(!parent_in(INT_MIN, i) && !parent_in(INT_MAX, i), "far parents", i);
    }
}

int main()
{
    masks();
    spans();
    std::printf("all passed\n");
    return 0;
}
