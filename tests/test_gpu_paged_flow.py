"""The paged KV cache's operators as a serving loop uses them: a model's prompt
moved into pages, tokens appended, read, weighed and evicted; in captured
graphs, on other streams, far into a large pool; and what they do with page
tables, lengths and row counts that they cannot follow."""
import os
import subprocess

import numpy as np
import pytest

from hip import Graph, Stream, copy
from nutllm_amd import workloads as W
from paged_case import Case, same

pytestmark = pytest.mark.gpu


def query_of(case, heads, seed=1):
    rng = np.random.default_rng(seed)
    return rng.standard_normal((case.batch, heads, case.dim)).astype(np.float32)


def near(case, heads, query, got, **kw):
    out, lse, weights, tol, _ = case.expect_attention(query, heads, **kw)
    assert np.all(np.abs(got - out) <= tol)
    return weights


def test_prompt_into_pages(gpu):
    """nut_prefill's K and V rows, layer by layer, behind what a sequence
    holds; attention over them."""
    cfg = W.make_config("step_gqa2", max_seq=96)
    model = W.build("step_gqa2", 0, 3, 96)
    dev, cache = model.to_device(), gpu.KVCache(cfg)
    dev.prefill(cache, W.synth_tokens(5, cfg.vocab_size, 70))
    keys, values = cache.read_positions(0, 70)
    for layer in range(cfg.layers):
        for begin, end in ((0, 70), (9, 42), (70, 70)):
            case = Case("f32", [5], cfg.kv_heads, cfg.head_dim, 16, seed=layer, room=70).upload()
            new = case.expect_append(keys[layer, :, begin:end].transpose(1, 0, 2),
                                     values[layer, :, begin:end].transpose(1, 0, 2),
                                     [end - begin])
            case.paged.append_cache(case.seqs, cache, layer, begin, end, case.d["new_lengths"],
                                    history=case.history)
            gpu.synchronize()
            assert np.array_equal(case.new_lengths(), new)
            for name in ("keys", "values"):
                assert same(case.pool(name), getattr(case, name))
            for name in ("bounds", "weights", "positions"):
                assert same(case.fetch(name), getattr(case, name))
            case.d["lengths"].upload(new)
            case.lengths = new
            q = query_of(case, 4)
            near(case, 4, q, case.attention(q, 4)[0])
    for layer, begin, end in ((cfg.layers, 0, 1), (0, 5, 4), (0, 0, 71)):
        with pytest.raises(gpu.OutOfRange):
            case.paged.append_cache(case.seqs, cache, layer, begin, end)
    other = Case("f32", [5], cfg.kv_heads + 1, cfg.head_dim, 16, room=70).upload()
    with pytest.raises(gpu.InvalidArgument, match="cache configuration mismatch"):
        other.paged.append_cache(other.seqs, cache, 0, 0, 1)
    cache.close(), dev.close()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_serving_loop(gpu, kind):
    """Ragged prompts, then tokens one at a time: append, attention that
    gathers weights, and an eviction to the budget whenever a sequence passes
    it; the host follows with the device's weights, which decide."""
    budget, heads, kv, dim = 40, 8, 2, 64
    case = Case(kind, [0, 0, 0], kv, dim, 16, seed=41, max_length=budget + 60).upload()
    case.bounds[:] = 0
    case.upload()
    rng, A = np.random.default_rng(7), gpu.DeviceArray
    counts, text = [50, 1, 37], np.zeros(3, np.int32)
    for step in range(14):
        rows = sum(counts)
        k = rng.standard_normal((rows, kv, dim)).astype(np.float32)
        v = rng.standard_normal((rows, kv, dim)).astype(np.float32)
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        new = case.expect_append(k, v, counts, firsts=text)
        case.paged.append(case.seqs, A(like=k), A(like=v), case.d["new_lengths"],
                          starts=A(like=starts) if step == 0 else None, max_new=max(counts),
                          history=case.history, first_positions=A(like=text))
        gpu.synchronize()
        assert np.array_equal(case.new_lengths(), new)
        text += np.array(counts, np.int32)
        case.lengths = new
        case.d["lengths"].upload(new)
        q = query_of(case, heads, step)
        grown = near(case, heads, q, case.attention(q, heads, history=case.history)[0])
        weights = case.fetch("weights")
        assert np.allclose(weights, case.weights + grown, rtol=1e-4, atol=1e-6)
        case.weights = weights
        if np.any(new > budget):
            new = case.expect_evict(budget, 2, 8)
            case.evict(budget, 2, 8)
            assert np.array_equal(case.new_lengths(), new)
            case.lengths = new
            case.d["lengths"].upload(new)
        for name in ("weights", "positions", "bounds"):
            assert same(case.fetch(name), getattr(case, name)), name
        for name in ("keys", "values"):
            assert same(case.pool(name), getattr(case, name)), name
        chosen = case.select(q, heads, 2, 0, 1)
        assert np.array_equal(chosen, case.expect_select(q, heads, 2, 0, 1))
        near(case, heads, q, case.attention(q, heads, selected=chosen, top=2)[0], selected=chosen)
        counts = [1, 1, 1]
    case.paged.check()


@pytest.mark.parametrize("prompts", [[40, 23], [90, 48]])
def test_new_tokens_stay_through_evictions(gpu, prompts):
    """Append, weigh and evict for more steps than the budget has rows, with the
    text's positions: what stays is the host's choice by the device's weights,
    the newest `last` tokens of every sequence are always there, and no position
    repeats."""
    budget, first, last, heads, kv, dim = 48, 2, 12, 4, 2, 16
    case = Case("f32", [0, 0], kv, dim, 8, seed=71, max_length=100)
    case.bounds[:] = 0
    case.upload()
    rng, A = np.random.default_rng(72), gpu.DeviceArray
    counts, text = prompts, np.zeros(2, np.int32)
    positions = A(like=text)
    for step in range(budget + 12):
        k, v = (rng.standard_normal((sum(counts), kv, dim)).astype(np.float32) for _ in range(2))
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        positions.upload(text)
        new = case.expect_append(k, v, counts, firsts=text)
        case.paged.append(case.seqs, A(like=k), A(like=v), case.d["new_lengths"],
                          starts=A(like=starts) if step == 0 else None, max_new=max(counts),
                          history=case.history, first_positions=positions)
        gpu.synchronize()
        text += np.array(counts, np.int32)
        case.lengths = new
        case.d["lengths"].upload(new)
        case.attention(query_of(case, heads, step), heads, history=case.history)
        case.weights = case.fetch("weights")
        new = case.expect_evict(budget, first, last)
        case.evict(budget, first, last)
        assert np.array_equal(case.new_lengths(), new)
        case.lengths = new
        case.d["lengths"].upload(new)
        for name in ("weights", "positions", "bounds"):
            assert same(case.fetch(name), getattr(case, name)), name
        for name in ("keys", "values"):
            assert same(case.pool(name), getattr(case, name)), name
        at = case.fetch("positions")
        for b in range(2):
            for h in range(kv):
                there = set(at[b, h, :new[b]].tolist())
                assert len(there) == new[b]
                assert there >= set(range(max(0, text[b] - last), text[b])), (step, b, h)
        counts = [1, 1]
    case.paged.check()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim,page,order", [
    (6, 2, 72, 16, "phs"), (12, 4, 104, 8, "psh"), (5, 5, 200, 32, "hps"), (40, 2, 16, 64, "sph"),
])
def test_views_with_room_between(gpu, kind, heads, kv, dim, page, order):
    """Rows with gaps between them, heads, slots and pages in any order, tables,
    queries and histories wider than they have to be, a table that two
    sequences of one length share: append, weigh, select, read and evict, what
    lies between left as it was."""
    lengths = [130, 1, 0, 77, 64]
    case = Case(kind, lengths, kv, dim, page, seed=91, room=3)
    # element strides, innermost axis last, each with room of 8 to 24 elements
    count, stride, at = dict(p=case.pages, h=kv, s=page), {}, dim + 8
    for i, axis in enumerate(reversed([a for a in order if a in count])):
        stride[axis], at = at, at * count[axis] + 8 * (i + 1)
    index = (np.arange(case.pages)[:, None, None, None] * stride["p"] +
             np.arange(kv)[:, None, None] * stride["h"] +
             np.arange(page)[:, None] * stride["s"] + np.arange(dim))
    A, flat = gpu.DeviceArray, {}
    for name in ("keys", "values"):
        flat[name] = np.full(at, 9, getattr(case, name).dtype)
        flat[name][index] = getattr(case, name)
    wide, span = case.width + 3, case.max_length + 5
    table = np.full((5, wide), -1, np.int32)
    table[:, :case.width] = case.table
    weights, positions = np.full((5, kv, span), 5.0, np.float32), np.full((5, kv, span), 6, np.int32)
    weights[..., :case.max_length], positions[..., :case.max_length] = case.weights, case.positions
    d = {name: A(like=x) for name, x in flat.items()}
    d.update(bounds=A(like=case.bounds), table=A(like=table), lengths=A(like=case.lengths),
             new=A(4 * 5), weights=A(like=weights), positions=A(like=positions),
             status=A(like=np.zeros(1, np.int32)))
    paged = gpu.PagedKV(d["keys"], d["values"], case.pages, page, kv, dim,
                        {"f32": gpu.F32, "f16": gpu.F16, "bf16": gpu.BF16}[kind],
                        strides=tuple(stride[a] for a in "phs"), bounds=d["bounds"],
                        status=d["status"])
    before, after = (gpu.PagedBatch(d["table"], wide, d[n], 5, case.max_length)
                     for n in ("lengths", "new"))
    history = gpu.PagedHistory(d["weights"], d["positions"], span)

    def compare():
        gpu.synchronize()
        for name in ("keys", "values"):
            flat[name][index] = getattr(case, name)
            assert same(d[name].download(flat[name].dtype, at), flat[name]), name
        assert same(d["bounds"].download(case.bounds.dtype, case.bounds.size),
                    case.bounds.reshape(-1))
        for name, want in (("weights", weights), ("positions", positions)):
            want[..., :case.max_length] = getattr(case, name)
            assert same(d[name].download(want.dtype, want.size).reshape(want.shape), want), name

    rows, counts, firsts = 8, [1, 3, 0, 2, 2], np.array([400, 1, 0, 77, 90], np.int32)
    k, v = (case.rng.standard_normal((rows, kv, dim)).astype(np.float32) for _ in range(2))
    starts = A(like=np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
    case.lengths = case.expect_append(k, v, counts, firsts=firsts)
    paged.append(before, A(like=k), A(like=v), d["new"], starts=starts, max_new=3, history=history,
                 first_positions=A(like=firsts))
    compare()
    room = heads * dim + 12
    query = np.full((5, room), np.nan, np.float32)
    query[:, :heads * dim] = query_of(case, heads).reshape(5, -1)
    q, out, space = A(like=query), A(4 * 5 * heads * dim), A(1 << 22)
    q64 = query[:, :heads * dim].reshape(5, heads, dim)

    def result():
        gpu.synchronize()
        return out.download(np.float32, 5 * heads * dim).reshape(5, heads, dim)

    assert paged.attention_workspace(after, heads, weighted=True) <= space.nbytes
    paged.attention(after, q, out, heads, query_stride=room, history=history, workspace=space)
    grown = near(case, heads, q64, result())
    got = d["weights"].download(np.float32, weights.size).reshape(weights.shape)
    assert np.allclose(got[..., :case.max_length], case.weights + grown, rtol=1e-4, atol=1e-6)
    case.weights = got[..., :case.max_length].copy()
    top, chosen = 3, A(4 * 5 * kv * 3)
    paged.select(after, q, chosen, heads, top, query_stride=room, workspace=space)
    want = case.expect_select(q64, heads, top, 1, 1)
    gpu.synchronize()
    assert np.array_equal(chosen.download(np.int32, want.size).reshape(want.shape), want)
    paged.attention(after, q, out, heads, query_stride=room, selected=chosen, top=top,
                    workspace=space)
    near(case, heads, q64, result(), selected=want)
    case.lengths = case.expect_evict(70, 2, 9)
    paged.evict(after, history, d["lengths"], 70, first=2, last=9, workspace=space)
    compare()
    assert np.array_equal(d["lengths"].download(np.int32, 5), case.lengths)
    paged.attention(before, q, out, heads, query_stride=room, workspace=space)
    near(case, heads, q64, result())
    # sequences that share pages which are only read
    table[1:] = table[0]
    d["table"].upload(table)
    case.table = np.tile(case.table[:1], (5, 1))
    case.lengths = np.array([70, 70, 30, 1, 0], np.int32)
    d["lengths"].upload(case.lengths)
    paged.attention(before, q, out, heads, query_stride=room, workspace=space)
    near(case, heads, q64, result())
    paged.check()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_many_short_sequences(gpu, kind):
    """A batch of 40,000 sequences, most of them of a row or none."""
    batch = 40000
    lengths = np.zeros(batch, np.int32)
    lengths[::37], lengths[5::1001], lengths[-1] = 1, 19, 19
    case = Case(kind, lengths[-1:], 1, 16, 8, seed=93, max_length=20)
    width, A = 3, gpu.DeviceArray
    # every sequence over the same three pages, which are only read
    seqs_table, d_lengths = A(like=np.tile(case.table, (batch, 1))), A(like=lengths)
    case.upload()
    seqs = gpu.PagedBatch(seqs_table, width, d_lengths, batch, 20)
    q = np.random.default_rng(4).standard_normal((batch, 2, 16)).astype(np.float32)
    dq, out, lse = A(like=q), A(q.nbytes), A(4 * batch * 2)
    chosen, space = A(4 * batch * 2), A(1 << 22)
    assert max(case.paged.attention_workspace(seqs, 2), case.paged.select_workspace(seqs, 2, 2)) \
        <= space.nbytes
    case.paged.attention(seqs, dq, out, 2, lse=lse, workspace=space)
    case.paged.select(seqs, dq, chosen, 2, 2, first=0, last=0, workspace=space)
    gpu.synchronize()
    got = out.download(np.float32, q.size).reshape(q.shape)
    none = lengths == 0
    assert np.all(got[none] == 0)
    assert np.all(np.isneginf(lse.download(np.float32, 2 * batch).reshape(batch, 2)[none]))
    value = case.rows(case.values, 0, 0)[0]
    # one row: its weight is 1, and 1 / 1
    assert np.all(np.abs(got[lengths == 1] - value) <= 2.0 ** -22 * np.abs(value))
    pages = chosen.download(np.int32, 2 * batch).reshape(batch, 2)
    assert np.all(pages[none] == -1) and np.all(pages[lengths == 1] == [0, -1])
    for b in np.flatnonzero(lengths == 19):
        one = Case(kind, [19], 1, 16, 8, seed=93, max_length=20)
        near(one, 2, q[b:b + 1], got[b:b + 1])
        assert np.array_equal(pages[b:b + 1, None], one.expect_select(q[b:b + 1], 2, 2, 0, 0))
    case.paged.check()


def test_captured_step(gpu):
    """A decode step (append, weighted attention, selection, attention over
    it, eviction) in two graphs with workspaces of their own, replayed in turn
    with other work between; each replay sees the inputs of its time."""
    heads, budget, top = 4, 100, 3
    case = Case("f16", [90, 130, 60], 2, 64, 16, seed=43, room=8).upload()
    A, stream, graphs = gpu.DeviceArray, Stream(), []
    k, v, q = A(4 * 3 * 2 * 64), A(4 * 3 * 2 * 64), A(4 * 3 * heads * 64)
    after = gpu.PagedBatch(case.d["table"], case.width, case.d["new_lengths"], 3, case.max_length)
    cut = A(like=np.zeros(3, np.int32))
    for _ in range(2):
        out, sparse, chosen = A(q.nbytes), A(q.nbytes), A(4 * 3 * 2 * top)
        sizes = (case.paged.attention_workspace(after, heads, weighted=True),
                 case.paged.select_workspace(after, heads, top),
                 case.paged.attention_workspace(after, heads, top=top),
                 case.paged.evict_workspace(after, budget))
        space = [A(like=np.full(max(1, n), 255, np.uint8)) for n in sizes]

        def step():
            at = stream.handle
            case.paged.append(case.seqs, k, v, case.d["new_lengths"], history=case.history,
                              stream=at)
            case.paged.attention(after, q, out, heads, history=case.history, workspace=space[0],
                                 stream=at)
            case.paged.select(after, q, chosen, heads, top, workspace=space[1], stream=at)
            case.paged.attention(after, q, sparse, heads, selected=chosen, top=top,
                                 workspace=space[2], stream=at)
            case.paged.evict(after, case.history, cut, budget, first=1, last=5,
                             workspace=space[3], stream=at)

        gpu.synchronize()
        graphs.append((Graph(stream, step), out, chosen, sparse, space))
    rng = np.random.default_rng(3)
    for turn in range(6):
        graph, out, chosen, sparse, _ = graphs[turn % 2]
        new = [rng.standard_normal(shape).astype(np.float32)
               for shape in ((3, 2, 64), (3, 2, 64), (3, heads, 64))]
        for array, x in zip((k, v, q), new):
            array.upload(x)
        gpu.synchronize()
        graph.replay()
        stream.synchronize()
        case.lengths = case.expect_append(new[0], new[1], [1, 1, 1])
        query = new[2]
        near(case, heads, query, out.download(np.float32, query.size).reshape(query.shape))
        want = case.expect_select(query, heads, top, 1, 1)
        assert np.array_equal(chosen.download(np.int32, want.size).reshape(want.shape), want)
        near(case, heads, query, sparse.download(np.float32, query.size).reshape(query.shape),
             selected=want)
        # the weights that decided, from the device: those below the budget
        # moved with their rows, so the plan is made from a copy of the state
        # before the move: the rows beyond the budget are where they were
        moved = case.fetch("weights")
        lengths = cut.download(np.int32, 3)
        assert np.array_equal(lengths, np.minimum(case.lengths, budget))
        at = case.fetch("positions")
        for b in range(3):
            n, m = int(case.lengths[b]), int(lengths[b])
            for h in range(2):
                there = {int(p): i for i, p in enumerate(case.positions[b, h, :n])}
                assert len({int(p) for p in at[b, h, :m]}) == m
                kept = [there[int(p)] for p in at[b, h, :m]]
                for i, j in enumerate(kept):
                    assert i == j or j >= budget
                    to, of = (case.table[b, x // 16] for x in (i, j))
                    for name in ("keys", "values"):
                        pool = getattr(case, name)
                        pool[to, h, i % 16] = pool[of, h, j % 16]
        case.weights, case.positions = moved, at
        case.bounds = case.fetch("bounds")
        for name in ("keys", "values"):
            assert same(case.pool(name), getattr(case, name)), name
        case.lengths = lengths
        case.d["lengths"].upload(lengths)
        gpu.synchronize()
    case.paged.check()
    for graph, *_ in graphs:
        graph.close()
    stream.close()


def test_captured_step_against_the_host(gpu):
    """A decode step captured with the text's positions and a copy of the
    weights between attention and eviction, replayed with other work between:
    positions, weights, bounds and rows are the host's choice by that copy, and
    the newest `last` tokens are there. Without first and last the same."""
    heads, budget, kv, dim = 4, 100, 2, 64
    A, stream = gpu.DeviceArray, Stream()
    rng = np.random.default_rng(74)
    for first, last in ((1, 5), (0, 0)):
        case = Case("f16", [90, 130, 60], kv, dim, 16, seed=73, room=8).upload()
        k, v, q = A(4 * 3 * kv * dim), A(4 * 3 * kv * dim), A(4 * 3 * heads * dim)
        after = gpu.PagedBatch(case.d["table"], case.width, case.d["new_lengths"], 3,
                               case.max_length)
        text = np.array([90, 130, 60], np.int32)
        positions, cut = A(like=text), A(like=np.zeros(3, np.int32))
        out, held = A(q.nbytes), A(like=case.weights)
        sizes = (case.paged.attention_workspace(after, heads, weighted=True),
                 case.paged.evict_workspace(after, budget))
        space = [A(like=np.full(max(1, n), 255, np.uint8)) for n in sizes]

        def step():
            at = stream.handle
            case.paged.append(case.seqs, k, v, case.d["new_lengths"], history=case.history,
                              first_positions=positions, stream=at)
            case.paged.attention(after, q, out, heads, history=case.history, workspace=space[0],
                                 stream=at)
            copy(held, case.d["weights"], stream)
            case.paged.evict(after, case.history, cut, budget, first=first, last=last,
                             workspace=space[1], stream=at)

        gpu.synchronize()
        graph = Graph(stream, step)
        for turn in range(6):
            new = [rng.standard_normal(shape).astype(np.float32)
                   for shape in ((3, kv, dim), (3, kv, dim), (3, heads, dim))]
            for array, x in zip((k, v, q, positions), (*new, text)):
                array.upload(x)
            gpu.synchronize()
            graph.replay()
            stream.synchronize()
            case.lengths = case.expect_append(new[0], new[1], [1, 1, 1], firsts=text)
            grown = near(case, heads, new[2],
                         out.download(np.float32, new[2].size).reshape(new[2].shape))
            text += 1
            weights = held.download(np.float32, case.weights.size).reshape(case.weights.shape)
            assert np.allclose(weights, case.weights + grown, rtol=1e-4, atol=1e-6)
            case.weights = weights
            case.lengths = case.expect_evict(budget, first, last)
            lengths = cut.download(np.int32, 3)
            assert np.array_equal(lengths, case.lengths)
            for name in ("weights", "positions", "bounds"):
                assert same(case.fetch(name), getattr(case, name)), name
            for name in ("keys", "values"):
                assert same(case.pool(name), getattr(case, name)), name
            at = case.fetch("positions")
            for b in range(3):
                for h in range(kv):
                    there = set(at[b, h, :lengths[b]].tolist())
                    assert len(there) == lengths[b]
                    assert there >= set(range(text[b] - last, text[b]))
            case.d["lengths"].upload(lengths)
            gpu.synchronize()
        graph.close()
        case.paged.check()
    stream.close()


def test_two_calls_at_once(gpu):
    """Calls on two streams with workspaces of their own."""
    case = Case("bf16", [900, 1500], 2, 64, 16, seed=45).upload()
    q = [query_of(case, 8, s) for s in (1, 2)]
    need = case.paged.attention_workspace(case.seqs, 8)
    work = [gpu.DeviceArray(like=np.full(max(1, need), 255, np.uint8)) for _ in q]
    dq = [gpu.DeviceArray(like=x) for x in q]
    out = [gpu.DeviceArray(4 * 2 * 8 * 64) for _ in q]
    streams = [Stream() for _ in q]
    gpu.synchronize()
    for _ in range(20):
        for s, a, o, w in zip(streams, dq, out, work):
            case.paged.attention(case.seqs, a, o, 8, workspace=w, stream=s.handle)
    for s in streams:
        s.synchronize()
    for x, o in zip(q, out):
        near(case, 8, x, o.download(np.float32, 2 * 8 * 64).reshape(2, 8, 64))


def test_same_answer_every_time(gpu):
    """Nothing depends on the order in which workgroups run."""
    case = Case("f16", [3000, 700], 2, 64, 16, seed=47).upload()
    q = query_of(case, 8)
    first = case.attention(q, 8)
    for _ in range(3):
        again = case.attention(q, 8)
        assert same(again[0], first[0]) and same(again[1], first[1])


@pytest.mark.parametrize("slot_major", [False, True])
def test_far_into_a_large_pool(gpu, slot_major):
    """Byte and element offsets beyond 32 bits: append, bounds, selection,
    attention and eviction with pages at both ends of a 12 GB pool."""
    kv, dim, ps, pages = 2, 64, 16, 1 << 20
    stride = kv * ps * dim + (64 if slot_major else 0)
    keys, values = (gpu.DeviceArray(4 * pages * stride) for _ in range(2))
    bounds = gpu.DeviceArray(4 * pages * kv * 2 * dim)
    strides = (stride, dim, kv * dim) if slot_major else (stride, ps * dim, dim)
    paged = gpu.PagedKV(keys, values, pages, ps, kv, dim, gpu.F32, strides=strides, bounds=bounds)
    table = np.array([[pages - 1, 0, pages // 2 + 1, pages - 2]], np.int32)
    case = Case("f32", [0], kv, dim, ps, seed=49, max_length=64)
    case.pages, case.table = 4, np.arange(4, dtype=np.int32)[None]
    n = 60
    k, v = (case.rng.standard_normal((n, kv, dim)).astype(np.float32) for _ in range(2))
    A = gpu.DeviceArray
    d_table, d_len, d_new = A(like=table), A(like=np.zeros(1, np.int32)), A(4)
    weights, positions = A(like=case.weights), A(like=case.positions)
    history = gpu.PagedHistory(weights, positions, 64)
    seqs = gpu.PagedBatch(d_table, 4, d_len, 1, 64)
    paged.append(seqs, A(like=k), A(like=v), d_new, starts=A(like=np.array([0, n], np.int32)),
                 max_new=n, history=history)
    case.lengths = case.expect_append(k, v, [n])
    after = gpu.PagedBatch(d_table, 4, d_new, 1, 64)
    q = query_of(case, 4)
    dq, out, chosen = A(like=q), A(4 * 4 * dim), A(4 * 2 * kv)
    space = A(1 << 20)
    paged.select(after, dq, chosen, 4, 2, first=0, last=1, workspace=space)
    paged.attention(after, dq, out, 4, selected=chosen, top=2, workspace=space)
    gpu.synchronize()
    want = case.expect_select(q, 4, 2, 0, 1)
    assert np.array_equal(chosen.download(np.int32, 2 * kv).reshape(1, kv, 2), want)
    near(case, 4, q, out.download(np.float32, 4 * dim).reshape(1, 4, dim), selected=want)
    paged.attention(after, dq, out, 4, workspace=space)
    gpu.synchronize()
    near(case, 4, q, out.download(np.float32, 4 * dim).reshape(1, 4, dim))
    case.weights = case.rng.random(case.weights.shape).astype(np.float32)
    weights.upload(case.weights)
    case.lengths = case.expect_evict(20)
    paged.evict(after, history, d_len, 20, workspace=space)
    paged.attention(seqs, dq, out, 4, workspace=space)
    gpu.synchronize()
    near(case, 4, q, out.download(np.float32, 4 * dim).reshape(1, 4, dim))


@pytest.mark.parametrize("bad", [-1, 1 << 30, 9])
def test_pages_that_the_cache_has_not(gpu, bad):
    """A bad entry's rows count nothing and are not written; entries behind a
    sequence's end are not read; the call says so once."""
    case = Case("f32", [40, 40], 1, 32, 16, seed=51, max_length=64, spare=1).upload()
    assert case.pages == 9
    q = query_of(case, 2)
    table = case.table.copy()
    table[0, 1] = bad     # rows 16 to 31
    table[:, 3] = bad     # behind the end: no matter
    case.d["table"].upload(table)
    got, lse = case.attention(q, 2)
    out, want_lse, _, tol, _ = case.expect_attention(q, 2)
    assert np.all(np.abs(got[1] - out[1]) <= tol[1])
    few = Case("f32", [40, 40], 1, 32, 16, seed=51, max_length=64, spare=1)
    rows = np.r_[0:16, 32:40]
    k, v = few.rows(few.keys, 0, 0)[rows], few.rows(few.values, 0, 0)[rows]
    for h in range(2):
        s = k @ q[0, h].astype(np.float64) * 32 ** -0.5
        p = np.exp(s - s.max())
        assert np.all(np.abs(got[0, h] - (p / p.sum()) @ v) <= 1e-5)
    with pytest.raises(gpu.OutOfRange, match="page out of range"):
        case.paged.check()
    case.paged.check()  # said once
    # a selection does not choose it before a page that there is
    table[0, 0] = bad
    case.d["table"].upload(table)
    assert case.select(q, 2, 1, 0, 0)[0, 0].tolist() == [2]
    with pytest.raises(gpu.OutOfRange, match="page out of range"):
        case.paged.check()
    # rows to be appended or moved there are left out; the others arrive
    case.d["table"].upload(case.table)
    before = case.pool("keys").copy()
    table = case.table.copy()
    table[0, 2] = bad
    case.d["table"].upload(table)
    ones = gpu.DeviceArray(like=np.ones((2, 1, 32), np.float32))
    case.paged.append(case.seqs, ones, ones, case.d["new_lengths"])
    gpu.synchronize()
    before[case.table[1, 2], 0, 8] = 1.0
    assert same(case.pool("keys"), before)
    case.evict(30)
    with pytest.raises(gpu.OutOfRange, match="page out of range"):
        case.paged.check()


def test_append_counts_rows_of_a_page_that_the_cache_has_not(gpu):
    """Rows on it are dropped; the new lengths, weights and positions are as if
    they were there, rows on the pages beside it arrive, and attention passes
    the missing ones over."""
    case = Case("f32", [10, 3], 2, 32, 16, seed=89, max_length=64).upload()
    k, v = (case.rng.standard_normal((45, 2, 32)).astype(np.float32) for _ in range(2))
    table = case.table.copy()
    table[0, 1] = case.pages  # rows 16 to 31
    case.d["table"].upload(table)
    missing = case.table[0, 1]
    before = [getattr(case, name)[missing].copy() for name in ("keys", "values", "bounds")]
    new = case.expect_append(k, v, [40, 5], firsts=[70, 7])
    for name, old in zip(("keys", "values", "bounds"), before):
        getattr(case, name)[missing] = old
    A = gpu.DeviceArray
    case.paged.append(case.seqs, A(like=k), A(like=v), case.d["new_lengths"],
                      starts=A(like=np.array([0, 40, 45], np.int32)), max_new=40,
                      history=case.history, first_positions=A(like=np.array([70, 7], np.int32)))
    gpu.synchronize()
    assert np.array_equal(case.new_lengths(), new)
    for name in ("weights", "positions", "bounds"):
        assert same(case.fetch(name), getattr(case, name)), name
    for name in ("keys", "values"):
        assert same(case.pool(name), getattr(case, name)), name
    with pytest.raises(gpu.OutOfRange, match="page out of range"):
        case.paged.check()
    case.lengths = new
    case.d["lengths"].upload(new)
    q = query_of(case, 4)
    got, _ = case.attention(q, 4)
    rows = np.r_[0:16, 32:50]
    for h in range(4):
        x, y = (case.rows(p, 0, h // 2)[rows] for p in (case.keys, case.values))
        s = x @ q[0, h].astype(np.float64) * 32 ** -0.5
        p = np.exp(s - s.max())
        # a score errs by (dim + 4) 2^-24 sum |q k|, below 2^-14; both parts by as much
        assert np.all(np.abs(got[0, h] - (p / p.sum()) @ y) <= 2.0 ** -12 * np.abs(y).max())
    with pytest.raises(gpu.OutOfRange, match="page out of range"):
        case.paged.check()


def test_lengths_and_counts_out_of_range(gpu):
    """A length below zero or over max_length holds no rows; appends that do
    not fit leave a sequence as it is."""
    case = Case("f32", [20, 20, 20, 20], 1, 32, 16, seed=53, max_length=32).upload()
    q = query_of(case, 2)
    case.d["lengths"].upload(np.array([20, -1, 33, 0], np.int32))
    got, lse = case.attention(q, 2)
    assert np.all(got[1:] == 0) and np.all(np.isneginf(lse[1:])) and np.all(np.isfinite(lse[0]))
    with pytest.raises(gpu.OutOfRange, match="length out of range"):
        case.paged.check()
    assert np.all(case.select(q, 2, 4, 1, 1)[1:] == -1)
    with pytest.raises(gpu.OutOfRange, match="length out of range"):
        case.paged.check()
    case.evict(10)
    assert case.new_lengths().tolist() == [10, -1, 33, 0]
    with pytest.raises(gpu.OutOfRange, match="length out of range"):
        case.paged.check()
    case = Case("f32", [20, 20, 20, 20], 1, 32, 16, seed=53, max_length=32).upload()
    A, rows = gpu.DeviceArray, np.ones((40, 1, 32), np.float32)
    before = case.pool("keys").copy()
    for starts in ([0, 13, 13, 13, 13],   # 33 rows of at most 32
                   [0, -1, -1, -1, -1], [5, 4, 4, 4, 4], [0, 14, 14, 14, 14],
                   [38, 41, 41, 41, 41], [-3, 0, 0, 0, 0]):
        case.paged.append(case.seqs, A(like=rows), A(like=rows), case.d["new_lengths"],
                          starts=A(like=np.array(starts, np.int32)), max_new=13,
                          history=case.history)
        gpu.synchronize()
        assert case.new_lengths().tolist() == [20] * 4
        assert same(case.pool("keys"), before)
        with pytest.raises(gpu.OutOfRange, match="out of range"):
            case.paged.check()
    assert same(case.fetch("weights"), case.weights)


def test_allocates_nothing(gpu):
    case = Case("bf16", [300, 40], 2, 64, 16, seed=55, room=1).upload()
    q = gpu.DeviceArray(like=query_of(case, 4))
    out, rows = gpu.DeviceArray(4 * 2 * 4 * 64), gpu.DeviceArray(4 * 2 * 2 * 64)
    chosen, space = gpu.DeviceArray(4 * 2 * 2 * 3), gpu.DeviceArray(1 << 20)
    before = gpu.device_allocations()
    case.paged.append(case.seqs, rows, rows, case.d["new_lengths"], history=case.history)
    case.paged.attention(case.seqs, q, out, 4, history=case.history, workspace=space)
    case.paged.select(case.seqs, q, chosen, 4, 3, workspace=space)
    case.paged.attention(case.seqs, q, out, 4, selected=chosen, top=3, workspace=space)
    case.paged.evict(case.seqs, case.history, case.d["new_lengths"], 50, workspace=space)
    gpu.synchronize()
    assert gpu.device_allocations() == before


def test_weights_of_rows_on_a_missing_page(gpu):
    """Rows on a page that the cache has not gather nothing, whole tiles of
    them included, whatever the workspace held."""
    case = Case("bf16", [200], 2, 64, 64, seed=57, max_length=256).upload()
    table = case.table.copy()
    table[0, 1] = -1  # rows 64 to 127
    case.d["table"].upload(table)
    case.attention(query_of(case, 4), 4, history=case.history)
    got = case.fetch("weights")
    assert same(got[0, :, 64:128], case.weights[0, :, 64:128])
    grown = (got - case.weights)[0, :, :200].sum(1)
    assert np.all(np.abs(grown - 2) <= 1e-4)  # two heads a KV head, all their weight
    with pytest.raises(gpu.OutOfRange, match="page out of range"):
        case.paged.check()


def test_cpp_host_api(gpu):
    binary = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build",
                          "paged_api_test")
    assert os.path.exists(binary), "build first: make -C tests/cpp"
    r = subprocess.run([binary], capture_output=True, text=True, timeout=60)
    print(r.stdout, flush=True)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr
