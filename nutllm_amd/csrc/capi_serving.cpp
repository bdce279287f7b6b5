// capi_serving.cpp — the extern "C" entry points of draft trees, page pools and
// beam search declared in include/nutllm_hip.h: every argument that the host can
// see is checked here, before anything is launched.
#include <cmath>

#include "paged_checks.hpp"
#include "serving.hpp"

namespace {

using namespace nut::checks;
using nut::require;

// Whether two ranges of bytes share none; null has none.
bool disjoint(const void *a, double a_bytes, const void *b, double b_bytes)
{
    const double x = double(reinterpret_cast<uintptr_t>(a));
    const double y = double(reinterpret_cast<uintptr_t>(b));
    return a == nullptr || b == nullptr || x + a_bytes <= y || y + b_bytes <= x;
}

nut::DraftView draft_of(const nut_draft *d)
{
    require(d != nullptr, NUT_EINVAL, "draft tree: null pointer");
    require(d->batch != 0 && d->batch <= kMost && d->most != 0 && d->total <= kMost, NUT_EINVAL,
            "draft tree: invalid dimensions");
    require(d->most <= nut::kMostNodes, NUT_EINVAL, "draft tree: more than 1024 nodes");
    require(d->d_starts != nullptr || d->total == d->batch * d->most, NUT_EINVAL,
            "draft tree: as many nodes a sequence without starts");
    return nut::DraftView{d->d_starts, d->d_parents, d->d_mask, d->mask_stride,
                          uint32_t(d->total), uint32_t(d->most), uint32_t(d->batch),
                          d->d_status};
}

void need_mask(const nut::DraftView &d)
{
    require(d.mask != nullptr, NUT_EINVAL, "draft tree: null pointer");
    require(d.mask_stride >= (d.most + 31) / 32 && d.mask_stride <= kMost, NUT_EINVAL,
            "draft tree: masks shorter than the nodes");
}

// The sequences of a draft, of which no page is read.
nut::PagedSeqs lengths_of(const nut::DraftView &d, const nut_paged_batch *s)
{
    require(s != nullptr && s->d_lengths != nullptr, NUT_EINVAL, "paged cache: null pointer");
    require(s->batch == d.batch && s->max_length <= kMost - 4096, NUT_EINVAL,
            "paged cache: invalid batch");
    return nut::PagedSeqs{s->d_pages, s->d_lengths, uint32_t(s->table_stride), d.batch,
                          uint32_t(s->max_length)};
}

// `count` layers from `at` on, at most kMostLayers.
nut::PagedLayers layers_of(const nut_paged_kv *layers, size_t at, size_t count)
{
    nut::PagedLayers got{};
    got.count = uint32_t(std::min<size_t>(count - at, nut::kMostLayers));
    got.view = view_of(layers);
    for (uint32_t i = 0; i < got.count; i++) {
        const nut::PagedView v = view_of(layers + at + i), &w = got.view;
        require(v.pages == w.pages && v.page_size == w.page_size && v.kv_heads == w.kv_heads &&
                    v.head_dim == w.head_dim && v.type == w.type &&
                    v.page_stride == w.page_stride && v.head_stride == w.head_stride &&
                    v.slot_stride == w.slot_stride &&
                    (v.bounds == nullptr) == (w.bounds == nullptr),
                NUT_EINVAL, "paged cache: layers of different shapes");
        got.keys[i] = v.keys, got.values[i] = v.values, got.bounds[i] = v.bounds;
    }
    require(got.view.kv_heads <= 65535, NUT_EINVAL,
            "paged cache: more rows than one launch covers");
    return got;
}

// Checks every layer before the first is launched, then runs `body` on each
// launch's.
template <typename Body>
void each_launch(const nut_paged_kv *layers, size_t count, Body &&body)
{
    require(layers != nullptr && count != 0, NUT_EINVAL, "paged cache: no layers");
    for (size_t at = 0; at < count; at += nut::kMostLayers)
        (void)layers_of(layers, at, count);
    nut::ensure_device();
    for (size_t at = 0; at < count; at += nut::kMostLayers)
        body(layers_of(layers, at, count));
}

nut::PoolView pool_of(const nut_page_pool *p)
{
    require(p != nullptr && p->d_refs != nullptr, NUT_EINVAL, "page pool: null pointer");
    require(p->pages != 0 && p->pages <= kMost && p->page_size != 0 && p->page_size <= kMost,
            NUT_EINVAL, "page pool: invalid dimensions");
    return nut::PoolView{p->d_refs, uint32_t(p->pages), uint32_t(p->page_size), p->d_status};
}

nut::TableView table_of(const nut_page_table *t)
{
    require(t != nullptr && t->d_pages != nullptr && t->d_lengths != nullptr &&
                t->d_held != nullptr,
            NUT_EINVAL, "page pool: null pointer");
    require(t->batch != 0 && t->batch <= kMost && t->stride != 0 && t->stride <= kMost, NUT_EINVAL,
            "page pool: invalid table");
    return nut::TableView{t->d_pages, t->d_lengths, t->d_held, uint32_t(t->stride),
                          uint32_t(t->batch)};
}

// Fresh pages are numbered over all entries of a new table, in 32 bits.
nut::TableView new_table_of(const nut_page_table *t)
{
    const nut::TableView v = table_of(t);
    require(double(v.batch) * v.stride <= double(0xffffffffu), NUT_EINVAL,
            "page pool: invalid table");
    return v;
}

struct Range {
    const void *p;
    double bytes;
};

// Whether none of what a call writes shares memory with what it reads: workgroups
// read while others write.
template <size_t W, size_t R>
bool apart_from(const Range (&written)[W], const Range (&read)[R])
{
    for (const Range &w : written)
        for (const Range &r : read)
            if (!disjoint(w.p, w.bytes, r.p, r.bytes))
                return false;
    return true;
}
template <size_t W> bool apart_themselves(const Range (&written)[W])
{
    for (const Range &w : written)
        for (const Range &x : written)
            if (&w != &x && !disjoint(w.p, w.bytes, x.p, x.bytes))
                return false;
    return true;
}

double entries_bytes(const nut::TableView &t) { return double(t.batch) * t.stride * 4; }

void check_apart(const nut::PoolView &pool, const nut::TableView &from, const nut::TableView &to,
                 const int *parents, const int *gains, const int *copies)
{
    const double old = from.batch, now = to.batch;
    const Range table[] = {{from.pages, entries_bytes(from)}, {from.lengths, old * 4},
                           {from.held, old * 4}, {parents, now * 4}};
    const Range each[] = {{gains, now * 4}};
    const Range written[] = {{to.pages, entries_bytes(to)}, {to.lengths, now * 4},
                             {to.held, now * 4}, {copies, now * 12}};
    require(apart_from(written, table) && apart_from(written, each), NUT_EINVAL,
            "page pool: the new table overlaps what is read");
    require(apart_themselves(written), NUT_EINVAL, "page pool: the new table overlaps itself");
    const Range refs[] = {{pool.refs, double(pool.pages) * 4}};
    require(apart_from(refs, table) && apart_from(refs, written), NUT_EINVAL,
            "page pool: the counts overlap a table");
}

nut::BeamsView beams_of(const nut_beams *b)
{
    require(b != nullptr && b->d_scores != nullptr, NUT_EINVAL, "beam search: null pointer");
    require(b->requests != 0 && b->requests <= kMost && b->beams != 0, NUT_EINVAL,
            "beam search: invalid dimensions");
    require(b->beams <= nut::kMostBeams, NUT_EINVAL, "beam search: more than 64 beams");
    return nut::BeamsView{b->d_scores, b->d_lengths, b->d_ended, uint32_t(b->requests),
                          uint32_t(b->beams)};
}

void check_beams(const nut::BeamsView &from, const nut::BeamsView &to, size_t vocab)
{
    require(from.requests == to.requests, NUT_EINVAL, "beam search: states of different requests");
    require((from.lengths == nullptr) == (to.lengths == nullptr) &&
                (from.ended == nullptr) == (to.ended == nullptr),
            NUT_EINVAL, "beam search: both states keep lengths and ends, or neither");
    require(vocab != 0 && vocab <= nut::kMostVocab, NUT_EINVAL,
            "beam search: vocabulary must be 1 to 262144");
    require(double(from.requests) * from.beams <= double(kMost) &&
                double(to.requests) * to.beams <= double(kMost),
            NUT_EINVAL, "beam search: invalid dimensions");
}

} // namespace

extern "C" {

int nut_draft_mask(const nut_draft *draft, int *d_depths, void *stream)
{
    return nut::guarded([&]() {
        const nut::DraftView d = draft_of(draft);
        need_mask(d);
        require(d.parents != nullptr, NUT_EINVAL, "draft tree: null pointer");
        nut::ensure_device();
        nut::launch_draft_mask(d, d_depths, as_stream(stream));
    });
}

int nut_draft_accept(const nut_draft *draft, const nut_paged_batch *seqs, const int *d_tokens,
                     const int *d_chosen, int *d_path, size_t path_stride, int *d_counts,
                     int *d_last, int *d_new_lengths, void *stream)
{
    return nut::guarded([&]() {
        const nut::DraftView d = draft_of(draft);
        const nut::PagedSeqs s = lengths_of(d, seqs);
        require(d.parents != nullptr && d_tokens != nullptr && d_chosen != nullptr &&
                    d_path != nullptr && d_counts != nullptr,
                NUT_EINVAL, "draft tree: null pointer");
        require(path_stride >= d.most && path_stride <= kMost, NUT_EINVAL,
                "draft tree: paths shorter than the nodes");
        require(apart(d_new_lengths, s.lengths, s.batch, s.batch), NUT_EINVAL,
                "paged cache: new lengths must not be the lengths");
        nut::ensure_device();
        nut::launch_draft_accept(d, s, d_tokens, d_chosen, d_path, path_stride, d_counts, d_last,
                                 d_new_lengths, as_stream(stream));
    });
}

size_t nut_paged_tree_attention_workspace(const nut_paged_kv *kv, const nut_paged_batch *seqs,
                                          const nut_draft *draft, size_t heads)
{
    return bytes_or_error([&]() {
        const nut::PagedView v = view_of(kv);
        const nut::PagedSeqs s = seqs_of(v, seqs);
        const nut::DraftView d = draft_of(draft);
        require(s.batch == d.batch, NUT_EINVAL, "paged cache: invalid batch");
        return nut::plan_tree(v, s, d, heads_of(v, heads)).bytes;
    });
}

int nut_paged_tree_attention(const nut_paged_kv *kv, const nut_paged_batch *seqs,
                             const nut_draft *draft, const float *d_query, size_t query_stride,
                             size_t heads, float scale, float *d_out, float *d_lse,
                             void *d_workspace, size_t workspace_bytes, void *stream)
{
    return nut::guarded([&]() {
        const nut::PagedView v = view_of(kv);
        const nut::PagedSeqs s = seqs_of(v, seqs);
        const nut::DraftView d = draft_of(draft);
        require(s.batch == d.batch, NUT_EINVAL, "paged cache: invalid batch");
        need_mask(d);
        const uint32_t n = heads_of(v, heads);
        query_stride = query_stride_of(v, d_query, query_stride, n);
        require(std::isfinite(scale), NUT_EINVAL, "paged attention: scale is not finite");
        require(d_out != nullptr, NUT_EINVAL, "paged cache: null pointer");
        require(aligned16(d_out), NUT_EINVAL,
                "paged cache: rows must start at multiples of 16 bytes");
        check_workspace(d_workspace, workspace_bytes, nut::plan_tree(v, s, d, n).bytes);
        nut::ensure_device();
        nut::launch_tree_attention(v, s, d, d_query, query_stride, n, scale, d_out, d_lse,
                                   static_cast<char *>(d_workspace), as_stream(stream));
    });
}

int nut_paged_keep(const nut_paged_kv *layers, size_t count, const nut_paged_batch *seqs,
                   const int *d_path, size_t path_stride, const int *d_counts, void *stream)
{
    return nut::guarded([&]() {
        require(layers != nullptr && count != 0, NUT_EINVAL, "paged cache: no layers");
        const nut::PagedSeqs s = seqs_of(view_of(layers), seqs);
        require(d_path != nullptr && d_counts != nullptr, NUT_EINVAL, "paged cache: null pointer");
        require(path_stride != 0 && path_stride <= kMost, NUT_EINVAL,
                "draft tree: paths shorter than the nodes");
        nut::paged_grid(uint64_t(s.batch) * layers->kv_heads *
                            std::min<size_t>(count, nut::kMostLayers), 64);
        each_launch(layers, count, [&](const nut::PagedLayers &l) {
            nut::launch_paged_keep(l, s, d_path, path_stride, d_counts, as_stream(stream));
        });
    });
}

size_t nut_pages_reorder_workspace(const nut_page_pool *pool, const nut_page_table *from,
                                   const nut_page_table *to)
{
    return bytes_or_error(
        [&]() { return nut::reorder_workspace(pool_of(pool), table_of(from), new_table_of(to)); });
}

int nut_pages_reorder(const nut_page_pool *pool, const nut_page_table *from,
                      const nut_page_table *to, const int *d_parents, const int *d_gains,
                      size_t gain, int *d_copies, void *d_workspace, size_t workspace_bytes,
                      void *stream)
{
    return nut::guarded([&]() {
        const nut::PoolView p = pool_of(pool);
        const nut::TableView old = table_of(from), now = new_table_of(to);
        require(d_parents != nullptr && d_copies != nullptr, NUT_EINVAL,
                "page pool: null pointer");
        require(gain <= kMost, NUT_EINVAL, "page pool: invalid gain");
        check_apart(p, old, now, d_parents, d_gains, d_copies);
        check_workspace(d_workspace, workspace_bytes, nut::reorder_workspace(p, old, now));
        nut::ensure_device();
        nut::launch_reorder(p, old, now, d_parents, d_gains, uint32_t(gain), d_copies,
                            static_cast<char *>(d_workspace), as_stream(stream));
    });
}

size_t nut_pages_compact_workspace(const nut_page_pool *pool, const nut_page_table *table)
{
    return bytes_or_error([&]() { return nut::compact_workspace(pool_of(pool), table_of(table)); });
}

int nut_pages_compact(const nut_page_pool *pool, const nut_page_table *table, size_t limit,
                      int *d_copies, size_t copies, void *d_workspace, size_t workspace_bytes,
                      void *stream)
{
    return nut::guarded([&]() {
        const nut::PoolView p = pool_of(pool);
        const nut::TableView t = table_of(table);
        require(limit <= p.pages, NUT_EINVAL, "page pool: limit beyond the pages");
        require(d_copies != nullptr, NUT_EINVAL, "page pool: null pointer");
        require(copies != 0 && copies <= kMost / 3, NUT_EINVAL, "page pool: invalid copies");
        const Range read[] = {{t.held, double(t.batch) * 4}};
        const Range written[] = {{p.refs, double(p.pages) * 4}, {t.pages, entries_bytes(t)},
                                 {d_copies, double(copies) * 12}};
        require(apart_from(written, read) && apart_themselves(written), NUT_EINVAL,
                "page pool: copies, counts and table overlap");
        check_workspace(d_workspace, workspace_bytes, nut::compact_workspace(p, t));
        nut::ensure_device();
        nut::launch_compact(p, t, uint32_t(limit), d_copies, uint32_t(copies),
                            static_cast<char *>(d_workspace), as_stream(stream));
    });
}

int nut_paged_copy(const nut_paged_kv *layers, size_t count, const int *d_copies, size_t copies,
                   void *stream)
{
    return nut::guarded([&]() {
        require(copies <= kMost / 3, NUT_EINVAL, "page pool: invalid copies");
        require(d_copies != nullptr || copies == 0, NUT_EINVAL, "page pool: null pointer");
        each_launch(layers, count, [&](const nut::PagedLayers &l) {
            if (copies != 0)
                nut::launch_paged_copy(l, d_copies, uint32_t(copies), as_stream(stream));
        });
    });
}

size_t nut_beam_select_workspace(const nut_beams *from, const nut_beams *to, size_t vocab)
{
    return bytes_or_error([&]() {
        const nut::BeamsView old = beams_of(from), now = beams_of(to);
        check_beams(old, now, vocab);
        return nut::beam_workspace(old, now, uint32_t(vocab));
    });
}

int nut_beam_select(const nut_beams *from, const nut_beams *to, const void *d_logits, int type,
                    size_t row_stride, size_t vocab, int eos, float power, int *d_parents,
                    int *d_tokens, void *d_workspace, size_t workspace_bytes, void *stream)
{
    return nut::guarded([&]() {
        const nut::BeamsView old = beams_of(from), now = beams_of(to);
        check_beams(old, now, vocab);
        require(d_logits != nullptr && d_parents != nullptr && d_tokens != nullptr, NUT_EINVAL,
                "beam search: null pointer");
        require(type == NUT_F32 || type == NUT_F16 || type == NUT_BF16, NUT_EINVAL,
                "beam search: unknown type");
        if (row_stride == 0)
            row_stride = vocab;
        require(row_stride >= vocab && row_stride < (size_t(1) << 40), NUT_EINVAL,
                "beam search: rows overlap");
        require(reinterpret_cast<uintptr_t>(d_logits) % nut::paged_element(type) == 0, NUT_EINVAL,
                "beam search: misaligned logits");
        require(eos >= -1 && (eos < 0 || size_t(eos) < vocab), NUT_EINVAL,
                "beam search: token out of range");
        require(std::isfinite(power) && std::fabs(power) <= 16.0f, NUT_EINVAL,
                "beam search: power must be -16 to 16");
        require(power == 0.0f || old.lengths != nullptr, NUT_EINVAL,
                "beam search: no lengths to rank by");
        const double before = double(old.requests) * old.beams * 4;
        const double after = double(now.requests) * now.beams * 4;
        const Range read[] = {{old.scores, before}, {old.lengths, before}, {old.ended, before}};
        const Range rows[] = {{d_logits, (double(row_stride) * (before / 4 - 1) + double(vocab)) *
                                             double(nut::paged_element(type))}};
        const Range written[] = {{now.scores, after}, {now.lengths, after}, {now.ended, after},
                                 {d_parents, after}, {d_tokens, after}};
        require(apart_from(written, read), NUT_EINVAL,
                "beam search: the new state overlaps the old one");
        require(apart_from(written, rows), NUT_EINVAL,
                "beam search: the new state overlaps the logits");
        require(apart_themselves(written), NUT_EINVAL,
                "beam search: the new state overlaps itself");
        check_workspace(d_workspace, workspace_bytes,
                        nut::beam_workspace(old, now, uint32_t(vocab)));
        nut::ensure_device();
        nut::launch_beam_select(old, now, d_logits, type, row_stride, uint32_t(vocab), eos, power,
                                d_parents, d_tokens, static_cast<char *>(d_workspace),
                                as_stream(stream));
    });
}

int nut_beam_gather(const void *d_from, size_t from_stride, size_t sources, void *d_to,
                    size_t to_stride, size_t rows, size_t row_bytes, const int *d_parents,
                    int *d_status, void *stream)
{
    return nut::guarded([&]() {
        require(d_from != nullptr && d_to != nullptr && d_parents != nullptr, NUT_EINVAL,
                "beam gather: null pointer");
        require(sources != 0 && sources <= kMost && rows != 0 && rows <= kMost && row_bytes != 0 &&
                    row_bytes < (size_t(1) << 40),
                NUT_EINVAL, "beam gather: invalid dimensions");
        if (from_stride == 0)
            from_stride = row_bytes;
        if (to_stride == 0)
            to_stride = row_bytes;
        require(from_stride < (size_t(1) << 40) && to_stride < (size_t(1) << 40), NUT_EINVAL,
                "beam gather: invalid dimensions");
        require((reinterpret_cast<uintptr_t>(d_from) | reinterpret_cast<uintptr_t>(d_to) |
                 from_stride | to_stride | row_bytes) % 4 == 0,
                NUT_EINVAL, "beam gather: rows must be multiples of 4 bytes");
        require(to_stride >= row_bytes || rows == 1, NUT_EINVAL, "beam gather: rows overlap");
        require(rows <= 0xffffffff / 256, NUT_EINVAL,
                "beam gather: more rows than one launch covers");
        require(disjoint(d_to, double(to_stride) * double(rows - 1) + double(row_bytes), d_from,
                         double(from_stride) * double(sources - 1) + double(row_bytes)),
                NUT_EINVAL, "beam gather: rows overlap");
        require(disjoint(d_to, double(to_stride) * double(rows - 1) + double(row_bytes), d_parents,
                         double(rows) * 4),
                NUT_EINVAL, "beam gather: the rows overlap the parents");
        nut::ensure_device();
        nut::launch_beam_gather(static_cast<const char *>(d_from), from_stride, uint32_t(sources),
                                static_cast<char *>(d_to), to_stride, uint32_t(rows), row_bytes,
                                d_parents, d_status, as_stream(stream));
    });
}

} // extern "C"
