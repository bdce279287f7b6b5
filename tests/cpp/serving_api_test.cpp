// serving_api_test.cpp — draft trees, page pools and beam search through the C++
// host API (include/nutllm_gpu.hpp): refusals with their exception types and
// messages, and on a GPU a tree verified, a table forked and a beam chosen, with
// results that are known by hand.
//
// usage: serving_api_test [--cpu-only]; exit status 0 when every check passes.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <stdexcept>
#include <vector>

#include "nutllm_gpu.hpp"

using namespace nutgpu;

namespace {

int failures = 0;

void report(bool ok, const char *name)
{
    std::printf("  %s %s\n", ok ? "ok" : "FAIL", name);
    if (!ok)
        failures++;
}

template <class E> bool throws(const std::function<void()> &f, const char *message)
{
    try {
        f();
    } catch (const E &e) {
        return std::strcmp(e.what(), message) == 0;
    } catch (...) {
        return false;
    }
    return false;
}

nut_paged_kv view_of(void *keys, void *values, int *status)
{
    nut_paged_kv v{};
    v.d_keys = keys, v.d_values = values;
    v.pages = 8, v.page_size = 4, v.kv_heads = 1, v.head_dim = 8;
    v.type = NUT_F32, v.d_status = status;
    return v;
}

void refusals()
{
    alignas(16) static int words[256];
    alignas(16) static float memory[64];
    int *word = words;
    const nut_draft tree{nullptr, 3, 3, 1, word, reinterpret_cast<unsigned *>(word), 1, nullptr};
    const nut_paged_batch seqs{word, 2, word, 1, 8};
    const PagedKV paged(view_of(memory, memory, word));
    nut_draft wide = tree;
    wide.most = wide.total = 1025;
    report(throws<std::invalid_argument>([&] { DraftTree(wide).build(); },
                                         "draft tree: more than 1024 nodes"),
           "a tree of too many nodes");
    report(throws<std::invalid_argument>([&] { paged.tree_attention_workspace(seqs, tree, 0); },
                                         "paged cache: heads must be a multiple of the KV heads"),
           "workspace of refused heads");
    report(throws<std::invalid_argument>(
               [&] { DraftTree(tree).accept(seqs, word, word, word, 2, word); },
               "draft tree: paths shorter than the nodes"),
           "short paths");
    report(throws<std::invalid_argument>([&] { PagedLayers({}).copy(word, 1); },
                                         "paged cache: no layers"),
           "no layers");
    const nut_page_table table{word, 4, word + 8, word + 16, 2};
    report(throws<std::invalid_argument>(
               [&] {
                   PagePool(nut_page_pool{word, 8, 4, nullptr})
                       .reorder(table, table, word + 24, nullptr, 1, word + 32, memory, 1 << 20);
               },
               "page pool: the new table overlaps what is read"),
           "a table in place");
    const nut_beams beams{memory, nullptr, nullptr, 1, 65};
    report(throws<std::invalid_argument>([&] { beam_select_workspace(beams, beams, 10); },
                                         "beam search: more than 64 beams"),
           "too many beams");
    report(throws<std::invalid_argument>([] { check_status_word(nullptr); },
                                         "paged cache: no status word"),
           "check without a status word");
}

template <typename T> std::vector<T> read(const DeviceBuffer &b, size_t count)
{
    std::vector<T> v(count);
    check(nut_memcpy_d2h(v.data(), b.get(), count * sizeof(T)));
    return v;
}

struct Ints : DeviceBuffer {
    explicit Ints(const std::vector<int> &v) : DeviceBuffer(v.size() * 4)
    {
        check(nut_memcpy_h2d(get(), v.data(), v.size() * 4));
    }
    int *p() const { return static_cast<int *>(get()); }
};

struct Floats : DeviceBuffer {
    explicit Floats(const std::vector<float> &v) : DeviceBuffer(v.size() * 4)
    {
        check(nut_memcpy_h2d(get(), v.data(), v.size() * 4));
    }
    float *p() const { return static_cast<float *>(get()); }
};

// Rows of zero keys, so that every row a node sees weighs the same; row i's value
// is i.
void device_checks()
{
    std::vector<float> zero(8 * 4 * 8, 0.0f), rows(8 * 4 * 8, 0.0f);
    for (int i = 0; i < 8; i++)
        for (int d = 0; d < 8; d++)
            rows[((i / 4 == 0 ? 5 : 2) * 4 + i % 4) * 8 + d] = float(i);
    const Floats keys(zero), values(rows), query(std::vector<float>(4 * 8, 1.0f)),
        out(std::vector<float>(4 * 8));
    const Ints status({0}), table({5, 2}), length({3}), parents({-1, 0, 0, 2}), mask({0, 0, 0, 0});
    const PagedKV paged(view_of(keys.get(), values.get(), status.p()));
    const nut_paged_batch seqs{table.p(), 2, length.p(), 1, 8};
    const nut_draft view{nullptr, 4, 4, 1, parents.p(), static_cast<unsigned *>(mask.get()), 1,
                         status.p()};
    const DraftTree tree(view);
    const Ints depths({9, 9, 9, 9}), tokens({7, 4, 6, 1}), chosen({6, 0, 1, 3}),
        path({-1, -1, -1, -1}), count({-1}), last({-1}), longer({-1});
    tree.build(depths.p());
    const size_t need = paged.tree_attention_workspace(seqs, view, 1);
    const DeviceBuffer work(need + 16);
    paged.tree_attention(seqs, view, query.p(), 1, 1.0f, out.p(), work.get(), need);
    tree.accept(seqs, tokens.p(), chosen.p(), path.p(), 4, count.p(), last.p(), longer.p());
    PagedLayers({paged.view()}).keep(seqs, path.p(), 4, count.p());
    check(nut_synchronize());
    report(read<int>(mask, 4) == std::vector<int>({1, 3, 5, 13}), "masks");
    report(read<int>(depths, 4) == std::vector<int>({0, 1, 1, 2}), "depths");
    // nodes are rows 3 to 6 behind rows 0, 1, 2
    const float want[] = {6 / 4.0f, 10 / 5.0f, 11 / 5.0f, 17 / 6.0f};
    const auto got = read<float>(out, 32);
    for (int i = 0; i < 4; i++)
        report(std::fabs(got[i * 8 + 3] - want[i]) < 1e-5f, "a node's mean");
    report(read<int>(path, 3) == std::vector<int>({0, 2, 3}) && read<int>(count, 1)[0] == 3 &&
               read<int>(last, 1)[0] == 3 && read<int>(longer, 1)[0] == 6,
           "the accepted path");
    const auto kept = read<float>(values, 8 * 4 * 8);
    report(kept[2 * 32 + 0] == 5.0f && kept[2 * 32 + 8] == 6.0f && kept[5 * 32 + 24] == 3.0f,
           "its rows");
    paged.check();

    // six rows of pages 5 and 2 become two sequences
    const Ints refs({0, 0, 1, 0, 0, 1, 0, 0}), six({6}), held({2}), both({0, 0}),
        pages({-1, -1, -1, -1}), lengths({0, 0}), holds({0, 0}), copies({0, 0, 0, 0, 0, 0});
    const nut_page_table now{table.p(), 2, six.p(), held.p(), 1},
        next{pages.p(), 2, lengths.p(), holds.p(), 2};
    const PagePool pool(nut_page_pool{refs.p(), 8, 4, status.p()});
    const size_t bytes = pool.reorder_workspace(now, next);
    const DeviceBuffer space(bytes);
    pool.reorder(now, next, both.p(), nullptr, 1, copies.p(), space.get(), bytes);
    PagedLayers({paged.view()}).copy(copies.p(), 2);
    check(nut_synchronize());
    report(read<int>(pages, 4) == std::vector<int>({5, 2, 5, 0}), "a forked table");
    report(read<int>(copies, 6) == std::vector<int>({-1, -1, -1, 2, 0, 2}), "the copy it asks for");
    report(read<int>(refs, 8) == std::vector<int>({1, 0, 1, 0, 0, 2, 0, 0}), "who holds what");
    report(read<float>(values, 8)[0] == 5.0f, "the copied row");
    check_status_word(status.p());

    // one beam, three tokens of logits 0, log 2, log 5: an eighth, a quarter, five eighths
    const Floats score({-1.0f}), logits({0.0f, std::log(2.0f), std::log(5.0f)}),
        scores({0.0f, 0.0f});
    const Ints parent({9, 9}), token({9, 9});
    const nut_beams from{score.p(), nullptr, nullptr, 1, 1}, to{scores.p(), nullptr, nullptr, 1, 2};
    const size_t room = beam_select_workspace(from, to, 3);
    const DeviceBuffer scratch(room);
    beam_select(from, to, logits.get(), NUT_F32, 3, -1, 0.0f, parent.p(), token.p(), scratch.get(),
                room);
    const Ints source({3, 4}), gathered({0, 0, 0, 0});
    beam_gather(source.get(), 1, gathered.get(), 2, 8, parent.p());
    check(nut_synchronize());
    const auto best = read<float>(scores, 2);
    report(read<int>(token, 2) == std::vector<int>({2, 1}) &&
               read<int>(parent, 2) == std::vector<int>({0, 0}),
           "the best tokens");
    report(std::fabs(best[0] - (-1.0f + std::log(0.625f))) < 1e-6f &&
               std::fabs(best[1] - (-1.0f + std::log(0.25f))) < 1e-6f,
           "their scores");
    report(read<int>(gathered, 4) == std::vector<int>({3, 4, 3, 4}), "the gathered rows");
}

} // namespace

int main(int argc, char **argv)
{
    refusals();
    if (!(argc > 1 && std::strcmp(argv[1], "--cpu-only") == 0))
        device_checks();
    if (failures == 0)
        std::printf("all passed\n");
    return failures == 0 ? 0 : 1;
}
