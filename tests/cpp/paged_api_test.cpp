// paged_api_test.cpp — the paged KV cache through the C++ host API
// (include/nutllm_gpu.hpp): refusals with their exception types and messages,
// and on a GPU a token appended, read, weighed, selected for and evicted, with
// rows whose results are known by hand.
//
// usage: paged_api_test [--cpu-only]; exit status 0 when every check passes.
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

nut_paged_kv view_of(void *keys, void *values, void *bounds, int *status)
{
    nut_paged_kv v{};
    v.d_keys = keys, v.d_values = values, v.d_bounds = bounds;
    v.pages = 4, v.page_size = 4, v.kv_heads = 1, v.head_dim = 8;
    v.type = NUT_F32, v.d_status = status;
    return v;
}

void refusals()
{
    int word = 0;
    alignas(16) static float memory[64];
    nut_paged_kv v = view_of(memory, memory, memory, &word);
    const nut_paged_batch seqs{&word, 2, &word, 1, 8};
    report(PagedKV(v).attention_workspace(seqs, 2) == 0, "one run needs no workspace");
    report(throws<std::invalid_argument>([&] { PagedKV(v).attention_workspace(seqs, 0); },
                                         "paged cache: heads must be a multiple of the KV heads"),
           "workspace of refused heads");
    report(throws<std::invalid_argument>(
               [&] { PagedKV(v).evict(seqs, {memory, &word, 8}, 4, 3, 2, &word + 1, memory, 256); },
               "paged evict: first and last rows exceed the budget"),
           "eviction that keeps more than its budget");
    report(throws<std::invalid_argument>(
               [&] { PagedKV(v).append(seqs, memory, memory, 0); },
               "paged append: one row a sequence without starts"),
           "append without rows");
    v.d_bounds = nullptr;
    report(throws<std::invalid_argument>(
               [&] { PagedKV(v).select(seqs, memory, 1, 1, 0, 1, &word, memory, 256); },
               "paged select: the cache keeps no bounds"),
           "selection without bounds");
    v.d_status = nullptr;
    report(throws<std::invalid_argument>([&] { PagedKV(v).check(); },
                                         "paged cache: no status word"),
           "check without a status word");
}

template <typename T> std::vector<T> read(const DeviceBuffer &b, size_t count)
{
    std::vector<T> v(count);
    check(nut_memcpy_d2h(v.data(), b.get(), count * sizeof(T)));
    return v;
}

template <typename T> void write(const DeviceBuffer &b, const std::vector<T> &v)
{
    check(nut_memcpy_h2d(b.get(), v.data(), v.size() * sizeof(T)));
}

// One sequence of six rows: row i has key (i, 0, ...) and value i everywhere.
void device_checks()
{
    const DeviceBuffer keys(4 * 4 * 8 * 4), values(4 * 4 * 8 * 4), bounds(4 * 2 * 8 * 4);
    const DeviceBuffer status(4), table(8), length(4), longer(4), cut(4), weights(32), at(32);
    const DeviceBuffer rows(6 * 8 * 4), vals(6 * 8 * 4), starts(8), query(2 * 8 * 4),
        out(2 * 8 * 4), lse(8), chosen(4), work(4096);
    write<int>(status, {0}), write<int>(table, {3, 1}), write<int>(length, {0});
    write<int>(starts, {0, 6});
    std::vector<float> k(48, 0.0f), v(48);
    for (int i = 0; i < 6; i++) {
        k[i * 8] = float(i);
        for (int d = 0; d < 8; d++)
            v[i * 8 + d] = float(i);
    }
    write(rows, k), write(vals, v);
    const PagedKV paged(view_of(keys.get(), values.get(), bounds.get(),
                                static_cast<int *>(status.get())));
    const nut_paged_history history{static_cast<float *>(weights.get()),
                                    static_cast<int *>(at.get()), 8};
    const auto seqs = [&](const DeviceBuffer &lengths) {
        return nut_paged_batch{static_cast<int *>(table.get()), 2,
                               static_cast<int *>(lengths.get()), 1, 8};
    };
    paged.append(seqs(length), static_cast<float *>(rows.get()), static_cast<float *>(vals.get()),
                 6, static_cast<int *>(starts.get()), 6, static_cast<int *>(longer.get()),
                 &history);
    check(nut_synchronize());
    report(read<int>(longer, 1)[0] == 6, "append gives the new length");

    // head 0 weighs row i by 3^i, head 1 all rows alike
    std::vector<float> q(16, 0.0f);
    q[0] = std::log(3.0f);
    write(query, q);
    const size_t need = paged.attention_workspace(seqs(longer), 2, 0, true);
    report(need <= 4096, "workspace fits");
    paged.attention(seqs(longer), static_cast<float *>(query.get()), 2, 1.0f,
                    static_cast<float *>(out.get()), work.get(), 4096,
                    static_cast<float *>(lse.get()), &history);
    check(nut_synchronize());
    const std::vector<float> o = read<float>(out, 16), l = read<float>(lse, 2);
    const double sum = 364.0; // 1 + 3 + ... + 243
    double mean = 0.0;
    for (int i = 0; i < 6; i++)
        mean += i * std::pow(3.0, i) / sum;
    report(std::fabs(o[0] - mean) < 1e-5 && o[7] == o[0] && std::fabs(o[8] - 2.5) < 1e-5,
           "attention of two heads");
    report(std::fabs(l[0] - std::log(sum)) < 1e-5 && std::fabs(l[1] - std::log(6.0)) < 1e-5,
           "log-sum-exp");
    const std::vector<float> w = read<float>(weights, 6);
    bool gathered = true;
    for (int i = 0; i < 6; i++)
        gathered = gathered &&
                   std::fabs(w[i] - (std::pow(3.0, i) / sum + 1.0 / 6)) < 1e-5;
    report(gathered, "weights of both heads");

    // the second page's keys are the larger ones
    paged.select(seqs(longer), static_cast<float *>(query.get()), 2, 1, 0, 0,
                 static_cast<int *>(chosen.get()), work.get(), 4096);
    check(nut_synchronize());
    report(read<int>(chosen, 1)[0] == 1, "the page of the largest keys");

    // rows 4 and 5 weigh most and move into the places of 1 and 2; 0 is kept
    paged.evict(seqs(longer), history, 3, 1, 0, static_cast<int *>(cut.get()), work.get(), 4096);
    check(nut_synchronize());
    report(read<int>(cut, 1)[0] == 3, "eviction gives the new length");
    const std::vector<int> p = read<int>(at, 3);
    report(p[0] == 0 && p[1] == 4 && p[2] == 5, "positions moved along");
    const std::vector<float> kept = read<float>(keys, 4 * 4 * 8);
    report(kept[3 * 32] == 0.0f && kept[3 * 32 + 8] == 4.0f && kept[3 * 32 + 16] == 5.0f,
           "keys moved");
    paged.check();

    write<int>(table, {4, 1});
    paged.attention(seqs(cut), static_cast<float *>(query.get()), 2, 1.0f,
                    static_cast<float *>(out.get()), work.get(), 4096);
    report(throws<std::out_of_range>([&] { paged.check(); }, "paged cache: page out of range"),
           "a page that the cache has not");
    report(read<float>(out, 1)[0] == 0.0f, "whose rows count nothing");
}

} // namespace

int main(int argc, char **argv)
{
    const bool cpu_only = argc > 1 && std::strcmp(argv[1], "--cpu-only") == 0;
    std::printf("paged KV cache checks\n");
    refusals();
    if (!cpu_only) {
        int devices = 0;
        if (nut_device_count(&devices) != NUT_OK || devices == 0) {
            std::printf("  FAIL no gfx950 device\n");
            return 1;
        }
        try {
            device_checks();
        } catch (const std::exception &e) {
            std::printf("  FAIL unexpected exception: %s\n", e.what());
            failures++;
        }
    }
    std::printf("%s\n", failures == 0 ? "all passed" : "FAILED");
    return failures == 0 ? 0 : 1;
}
