"""Draft trees, page pools and beams as a program uses them together: greedy
decoding that verifies drafted trees, beam search over forked pages, both against
plain host programs in 64 bits; many sequences, captured graphs, two streams."""
import os
import subprocess

import numpy as np
import pytest

import nutllm_amd as nut
from hip import Graph, Stream, copy
from paged_case import TYPES, decode, encode
from serving_case import TreeCase, beam_step, dev, path_of, space, tree_of

pytestmark = pytest.mark.gpu
HEADS, KV, DIM, VOCAB = 4, 2, 16, 31


class Toy:
    """One attention layer over tables of queries, keys and values by token and place;
    logits are the tokens' readings of its output."""

    def __init__(self, seed, kind):
        rng = np.random.default_rng(seed)
        self.kind = kind
        self.q = rng.standard_normal((VOCAB, HEADS, DIM)).astype(np.float32) * 2
        self.k = rng.standard_normal((VOCAB, KV, DIM)).astype(np.float32)
        self.v = rng.standard_normal((VOCAB, KV, DIM)).astype(np.float32)
        self.place = rng.standard_normal((64, KV, DIM)).astype(np.float32) * 0.5
        self.read = rng.standard_normal((HEADS * DIM, VOCAB)).astype(np.float32) * 3

    def rows(self, tokens, places):
        return self.k[tokens] + self.place[np.asarray(places) % 64], self.v[tokens]

    def logits(self, out):
        """fp32 logits of fp32 attention results [n][heads][dim]."""
        return (np.asarray(out, np.float64).reshape(-1, HEADS * DIM) @ self.read).astype(np.float32)

    def host(self, text):
        """Logits behind a text, in 64 bits, over rows as the cache's type keeps them."""
        k, v = self.rows(np.asarray(text), np.arange(len(text)))
        k, v = (decode(encode(a, self.kind), self.kind) for a in (k, v))
        out = np.zeros((HEADS, DIM))
        for h in range(HEADS):
            s = k[:, h // 2] @ self.q[text[-1], h].astype(np.float64) * DIM ** -0.5
            p = np.exp(s - s.max())
            out[h] = (p / p.sum()) @ v[:, h // 2]
        return out.reshape(-1) @ self.read.astype(np.float64)


class Cache:
    """A paged cache of one layer with a page pool, all on the device."""

    def __init__(self, kind, pages, page, width):
        shape = (pages, KV, page, DIM)
        rows = encode(np.full(shape, np.nan), kind)
        self.keys, self.values = nut.DeviceArray(like=rows), nut.DeviceArray(like=rows)
        self.bounds = nut.DeviceArray(like=encode(np.zeros((pages, KV, 2, DIM)), kind))
        self.status, self.refs = dev([0]), dev(np.zeros(pages))
        self.kv = nut.PagedKV(self.keys, self.values, pages, page, KV, DIM, TYPES[kind],
                              bounds=self.bounds, status=self.status)
        self.layers = nut.PagedLayers([self.kv])
        self.pool = nut.PagePool(self.refs, pages, page, status=self.status)
        self.page, self.width = page, width
        self.table = [dev(np.full((1, width), -1)), dev([0]), dev([0])]
        self.batch = 1

    def view(self):
        return nut.PageTable(self.table[0], self.width, self.table[1], self.table[2], self.batch)

    def step(self, parents, gain):
        """The next table, its pages copied where they part."""
        n = parents.nbytes // 4
        old = self.view()
        table = [dev(np.full((n, self.width), -1)), dev(np.zeros(n)), dev(np.zeros(n))]
        new = nut.PageTable(table[0], self.width, table[1], table[2], n)
        copies = dev(np.zeros((n, 3)))
        self.pool.reorder(old, new, parents, copies, gain=gain,
                          workspace=space(self.pool.reorder_workspace(old, new)))
        self.layers.copy(copies, n)
        nut.synchronize()
        self.table, self.batch = table, n

    def seqs(self):
        return nut.PagedBatch(self.table[0], self.width, self.table[1], self.batch,
                              self.width * self.page)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,nodes", [(4, 9), (16, 40), (1, 3)])
def test_greedy_decoding_by_trees(gpu, kind, page, nodes):
    """Texts grow by what the model agrees with of random trees, with the token that it
    chooses behind that; what comes out is what one token at a time gives."""
    toy, rng = Toy(page, kind), np.random.default_rng(nodes)
    prompts = [[3, 1, 4, 1, 5], [9], [2, 6, 5, 3, 5, 8, 9, 7]]
    batch = len(prompts)
    cache = Cache(kind, 600, page, 128 // page + nodes)
    cache.step(dev([-1] * batch), 10)
    # the prompts but for their last tokens, which are the first trees' roots
    starts = np.concatenate([[0], np.cumsum([len(p) - 1 for p in prompts])])
    k, v = toy.rows(np.concatenate([p[:-1] for p in prompts]).astype(int),
                    np.concatenate([np.arange(len(p) - 1) for p in prompts]))
    grown = dev(np.zeros(batch))
    cache.kv.append(cache.seqs(), dev(k, np.float32), dev(v, np.float32), grown,
                    starts=dev(starts), max_new=10)
    cache.table[1] = grown
    texts = [list(p) for p in prompts]
    accepted = 0
    for _ in range(7):
        cache.step(dev(np.arange(batch)), nodes)
        counts = [nodes, 1 + int(rng.integers(0, nodes)), nodes]
        starts = np.concatenate([[0], np.cumsum(counts)])
        total = int(starts[-1])
        parents = [tree_of(rng, m) for m in counts]
        tokens, places = np.zeros(total, int), np.zeros(total, int)
        for b, p in enumerate(parents):
            lines = [texts[b]]
            for i, parent in enumerate(p):
                line = lines[0] if parent < 0 else lines[parent + 1]
                if i == 0:
                    token = texts[b][-1]
                else:  # often what the model says, so that paths grow
                    token = int(np.argmax(toy.host(line))) if rng.random() < 0.6 else \
                        int(rng.integers(0, VOCAB))
                    line = line + [token]
                lines.append(line)
                tokens[starts[b] + i], places[starts[b] + i] = token, len(line) - 1
        flat = dev(np.concatenate(parents))
        mask, depths = dev(np.zeros((total, (nodes + 31) // 32)), np.uint32), dev(np.zeros(total))
        draft = nut.DraftTree(flat, mask, nodes, total, batch, starts=dev(starts),
                              status=cache.status)
        draft.build(depths=depths)
        depth = depths.download(np.int32, total)
        for b in range(batch):
            assert np.array_equal(places[starts[b]:starts[b + 1]],
                                  len(texts[b]) - 1 + depth[starts[b]:starts[b + 1]])
        k, v = toy.rows(tokens, places)
        behind = dev(np.zeros(batch))
        cache.kv.append(cache.seqs(), dev(k, np.float32), dev(v, np.float32), behind,
                        starts=dev(starts), max_new=nodes)
        out = dev(np.zeros((total, HEADS, DIM)), np.float32)
        need = cache.kv.tree_attention_workspace(cache.seqs(), draft, HEADS)
        cache.kv.tree_attention(cache.seqs(), draft, dev(toy.q[tokens], np.float32), out, HEADS,
                                workspace=space(need))
        logits = toy.logits(out.download(np.float32, total * HEADS * DIM))
        one = nut.BeamState(dev(np.zeros(total), np.float32), total, 1)
        best = nut.BeamState(dev(np.zeros(total), np.float32), total, 1)
        chosen = dev(np.zeros(total))
        nut.beam_select(one, best, dev(logits, np.float32), VOCAB, dev(np.zeros(total)), chosen,
                        workspace=space(nut.beam_select_workspace(one, best, VOCAB)))
        path, kept, last = dev(np.zeros((batch, nodes))), dev([0] * batch), dev([0] * batch)
        lengths = dev(np.zeros(batch))
        draft.accept(cache.seqs(), dev(tokens), chosen, path, kept, last=last, new_lengths=lengths)
        cache.layers.keep(cache.seqs(), path, nodes, kept)
        cache.table[1] = lengths
        gpu.check_status(cache.status)
        n = kept.download(np.int32, batch)
        way = path.download(np.int32, batch * nodes).reshape(batch, nodes)
        choice = chosen.download(np.int32, total)
        for b in range(batch):
            at = slice(starts[b], starts[b + 1])
            assert way[b, :n[b]].tolist() == path_of(parents[b], tokens[at], choice[at])
            texts[b] += tokens[at][way[b, 1:n[b]]].tolist() + [int(last.download(np.int32, batch)[b])]
            accepted += int(n[b]) - 1
    assert accepted > 5
    for b, prompt in enumerate(prompts):
        for i in range(len(prompt), len(texts[b])):
            x = toy.host(texts[b][:i])
            two = np.sort(x)[-2:]
            assert two[1] - two[0] > 1e-3, "the toy's choices are apart"
            assert texts[b][i] == int(np.argmax(x))
    # the rows are the text's, one behind another
    table = cache.table[0].download(np.int32, batch * cache.width).reshape(batch, -1)
    shape = (600, KV, page, DIM)
    dtype = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[kind]
    pools = [a.download(dtype, int(np.prod(shape))).reshape(shape)
             for a in (cache.keys, cache.values)]
    for b, text in enumerate(texts):
        i = np.arange(len(text) - 1)
        assert cache.table[1].download(np.int32, batch)[b] == len(i)
        for pool, rows in zip(pools, toy.rows(np.asarray(text[:-1]), i)):
            assert np.array_equal(pool[table[b, i // page], :, i % page], encode(rows, kind))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("page,power", [(4, 0.0), (16, 0.8)])
def test_beam_search(gpu, kind, page, power):
    """Two texts, three beams each, until some end: tokens, scores and lengths are those
    of a host program that keeps whole texts."""
    toy, eos, beams, requests = Toy(7 + page, kind), 5, 3, 2
    prompts = [[3, 1, 4, 1, 5, 9, 2], [6, 5]]
    cache = Cache(kind, 200, page, 128 // page)
    cache.step(dev([-1] * requests), 8)
    starts = np.concatenate([[0], np.cumsum([len(p) for p in prompts])])
    k, v = toy.rows(np.concatenate(prompts), np.concatenate([np.arange(len(p)) for p in prompts]))
    grown = dev(np.zeros(requests))
    cache.kv.append(cache.seqs(), dev(k, np.float32), dev(v, np.float32), grown,
                    starts=dev(starts), max_new=8)
    cache.table[1] = grown
    cache.step(dev(np.repeat(np.arange(requests), beams)), 1)
    n = requests * beams
    host = [[list(p)] * beams for p in prompts]
    scores = np.full((requests, beams), -np.inf)
    scores[:, 0] = 0.0
    lengths, ended = np.zeros((2, requests, beams), int)
    state = [dev(scores, np.float32), dev(lengths), dev(ended)]
    texts = dev(np.full((n, 40), -1))
    for step in range(12):
        last = [host[r][i][-1] for r in range(requests) for i in range(beams)]
        out = dev(np.zeros((n, HEADS, DIM)), np.float32)
        need = cache.kv.attention_workspace(cache.seqs(), HEADS)
        cache.kv.attention(cache.seqs(), dev(toy.q[last], np.float32), out, HEADS,
                           workspace=space(need))
        logits = toy.logits(out.download(np.float32, n * HEADS * DIM))
        exact = np.array([[toy.host(t) for t in row] for row in host])
        now = nut.BeamState(state[0], requests, beams, lengths=state[1], ended=state[2])
        new = [dev(np.zeros(n), np.float32), dev(np.zeros(n)), dev(np.zeros(n))]
        then = nut.BeamState(new[0], requests, beams, lengths=new[1], ended=new[2])
        parents, tokens = dev(np.zeros(n)), dev(np.zeros(n))
        nut.beam_select(now, then, dev(logits, np.float32), VOCAB, parents, tokens, eos=eos,
                        power=power, workspace=space(nut.beam_select_workspace(now, then, VOCAB)))
        more = dev(np.full((n, 40), -1))
        nut.beam_gather(texts, more, 160, parents, rows=n, sources=n, status=cache.status)
        cache.step(parents, 1)
        gpu.check_status(cache.status)
        (wp, wt, ws, wl, we), ranks = beam_step(scores, lengths, ended, exact, beams, eos, power)
        gap = -np.diff(ranks, axis=1)
        assert np.all((gap == 0) | (gap > 1e-4)), "the toy's beams are apart"
        assert np.array_equal(parents.download(np.int32, n).reshape(wp.shape), wp)
        assert np.array_equal(tokens.download(np.int32, n).reshape(wt.shape), wt)
        assert np.array_equal(new[1].download(np.int32, n).reshape(wl.shape), wl)
        assert np.array_equal(new[2].download(np.int32, n).reshape(we.shape), we)
        got = new[0].download(np.float32, n).reshape(ws.shape)
        assert np.all(np.abs(got - ws) < 1e-4)  # logits of fp32 rows, summed over the steps
        host = [[host[r][wp[r, i] - r * beams] +
                 ([] if ended.ravel()[wp[r, i]] else [int(wt[r, i])]) for i in range(beams)]
                for r in range(requests)]
        # the new tokens' rows, and the texts; ended beams append too, and are not read again
        k, v = toy.rows(wt.ravel(), np.array([len(t) - 1 for row in host for t in row]))
        grown = dev(np.zeros(n))
        cache.kv.append(cache.seqs(), dev(k, np.float32), dev(v, np.float32), grown)
        cache.table[1] = grown
        rows = more.download(np.int32, n * 40).reshape(n, 40)
        rows[np.arange(n), step] = np.where(ended.ravel()[wp.ravel()] != 0, -1, wt.ravel())
        texts = dev(rows)
        scores, lengths, ended, state = ws, wl, we, new
        for i, row in enumerate(rows):
            r, k = divmod(i, beams)
            assert row[row >= 0].tolist() == host[r][k][len(prompts[r]):]
    refs = cache.refs.download(np.int32, 200)
    table = cache.table[0].download(np.int32, n * cache.width)
    held = cache.table[2].download(np.int32, n)
    count = np.zeros(200, int)
    for b in range(n):
        np.add.at(count, table.reshape(n, -1)[b, :held[b]], 1)
    assert np.array_equal(refs, count)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim,order", [(8, 1, 64, False), (6, 2, 80, True),
                                                (2, 2, 128, False), (4, 1, 32, True),
                                                (4, 1, 256, False), (4, 2, 96, False),
                                                (3, 1, 8, False), (5, 1, 136, True)])
def test_many_query_rows(gpu, kind, heads, kv, dim, order):
    """Blocks of query rows with rows in shared memory: ragged trees, idle sequences, a
    table far wider than they need, shares that cut blocks anywhere."""
    held = [0, 700, 1, 33, 0, 257, 64, 63, 500, 5]
    counts = [90, 60, 33, 1, 0, 129, 64, 17, 3, 70]
    c = TreeCase(kind, held, counts, kv, dim, 16, heads, seed=dim, slot_major=order, lead=1,
                 max_length=9000, trail=2)
    c.upload().check()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_many_sequences_of_trees(gpu, kind):
    """More sequences than a workgroup has threads."""
    rng = np.random.default_rng(3)
    held = rng.integers(0, 60, 700).tolist()
    counts = np.where(rng.random(700) < 0.3, 0, rng.integers(1, 41, 700)).tolist()
    counts[0], counts[-1] = 0, 40
    TreeCase(kind, held, counts, 1, 16, 16, 1, seed=5, max_length=600).upload().check()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_unseen_rows_that_are_not_finite_beside_many_queries(gpu, kind):
    c = TreeCase(kind, [100, 0], [70, 90], 1, 64, 16, 2, seed=4, max_length=9000)
    out, lse, tol, tol_lse = c.expect()
    rows = {0: [(5, np.inf), (40, np.nan)], 1: [(33, -np.inf)]}
    for b, bad in rows.items():
        for i, x in bad:
            row = c.held[b] + i
            c.case.values[c.case.table[b, row // 16], 0, row % 16, 7] = encode(np.array([x]), kind)[0]
            c.case.keys[c.case.table[b, row // 16], 0, row % 16, 9] = encode(np.array([0.5]), kind)[0]
    out, lse, tol, tol_lse = TreeCase.expect(c)
    got, got_lse = c.upload().attention()
    for b, bad in rows.items():
        for i in range(c.counts[b]):
            at, seen = c.starts[b] + i, [x for j, x in bad if c.sees[b][i, j]]
            rest = np.arange(64) != 7
            assert np.all(np.abs(got[at][:, rest] - out[at][:, rest]) <= tol[at][:, rest])
            assert np.all(np.abs(got_lse[at] - lse[at]) <= tol_lse[at])
            if not seen:
                assert np.all(np.abs(got[at][:, 7] - out[at][:, 7]) <= tol[at][:, 7])
            elif len(set(map(str, seen))) == 1:
                assert np.all(np.isnan(got[at][:, 7]) if np.isnan(seen[0])
                              else got[at][:, 7] == seen[0])


def test_captured_verification(gpu):
    """Masks, attention, the path and its rows, captured: each replay gives what the
    eager calls gave, with other work on the device in between."""
    stream = Stream()
    c = TreeCase("bf16", [100, 3, 40], [40, 33, 7], 2, 64, 16, 8, seed=2, max_length=6000).upload()
    rng = np.random.default_rng(0)
    flat, total, batch = np.concatenate(c.parents), c.total, 3
    tokens, chosen = (dev(rng.integers(0, 2, total)) for _ in range(2))
    draft = gpu.DraftTree(dev(flat), c.d_mask, c.most, total, batch, starts=c.d_starts,
                          status=c.status)
    depths, path = dev(np.zeros(total)), dev(np.zeros((batch, c.most)))
    counts, last, new = (dev(np.zeros(batch)) for _ in range(3))
    out, lse = dev(np.zeros((total, 8, 64)), np.float32), dev(np.zeros((total, 8)), np.float32)
    work = space(c.case.paged.tree_attention_workspace(c.seqs, draft, 8))
    keys, values = c.case.d["keys"], c.case.d["values"]
    saved = [gpu.DeviceArray(nbytes=a.nbytes) for a in (keys, values)]
    layers = gpu.PagedLayers([c.case.paged])
    h = stream.handle
    copy(saved[0], keys, stream), copy(saved[1], values, stream)
    stream.synchronize()

    def work_of(s):
        draft.build(depths=depths, stream=s)
        c.case.paged.tree_attention(c.seqs, draft, c.d_query, out, 8, lse=lse, workspace=work,
                                    stream=s)
        draft.accept(c.seqs, tokens, chosen, path, counts, last=last, new_lengths=new, stream=s)
        layers.keep(c.seqs, path, c.most, counts, stream=s)

    buffers = [(out, np.uint32), (lse, np.uint32), (path, np.int32), (counts, np.int32),
               (last, np.int32), (new, np.int32), (keys, np.uint16), (values, np.uint16),
               (c.d_mask, np.uint32), (depths, np.int32)]

    def state():
        stream.synchronize()
        return [a.download(t, a.nbytes // np.dtype(t).itemsize) for a, t in buffers]

    work_of(h)
    want = state()
    assert want[3].max() > 1
    graph = Graph(stream, lambda: work_of(h))
    for k in range(4):
        copy(keys, saved[0], stream), copy(values, saved[1], stream)
        for a, t in buffers[:6]:
            # what stands behind a path stays: as it was for the eager calls
            a.upload(np.full(a.nbytes // 4, 0 if a is path else 99, np.uint32))
        if k % 2:
            TreeCase("f16", [30], [5], 1, 32, 16, 2, seed=k).upload().check()
        graph.replay()
        for got, w in zip(state(), want):
            assert np.array_equal(got, w)
    c.case.paged.check()
    graph.close(), stream.close()


def test_captured_beam_step(gpu):
    stream = Stream()
    rng = np.random.default_rng(1)
    requests, beams, vocab, pages, page, width = 3, 4, 5000, 80, 4, 6
    n, h = requests * beams, stream.handle
    logits = dev(rng.standard_normal((n, vocab)) * 3, np.float32)
    scores = dev(-rng.random(n) * 3, np.float32)
    new, parents, tokens = dev(np.zeros(n), np.float32), dev(np.zeros(n)), dev(np.zeros(n))
    old_state, new_state = (gpu.BeamState(a, requests, beams) for a in (scores, new))
    table = rng.permutation(pages)[:n * 3].reshape(n, 3)
    entries = np.full((n, width), -1)
    entries[:, :3] = table
    refs = np.zeros(pages)
    refs[table] = 1
    d_refs, kept_refs, status = dev(refs), dev(refs), dev([0])
    rows = encode(rng.standard_normal((pages, 2, page, 16)), "bf16")
    keys, values = gpu.DeviceArray(like=rows), gpu.DeviceArray(like=rows[::-1].copy())
    layers = gpu.PagedLayers([gpu.PagedKV(keys, values, pages, page, 2, 16, gpu.BF16,
                                          status=status)])
    pool = gpu.PagePool(d_refs, pages, page, status=status)
    old = gpu.PageTable(dev(entries), width, dev(np.full(n, 10)), dev(np.full(n, 3)), n)
    d = [dev(np.full((n, width), -1)), dev(np.zeros(n)), dev(np.zeros(n)), dev(np.zeros((n, 3)))]
    then = gpu.PageTable(d[0], width, d[1], d[2], n)
    work = space(gpu.beam_select_workspace(old_state, new_state, vocab))
    more = space(pool.reorder_workspace(old, then))
    text, moved = dev(rng.integers(0, 99, (n, 20))), dev(np.zeros((n, 20)))

    def step(s):
        gpu.beam_select(old_state, new_state, logits, vocab, parents, tokens, workspace=work,
                        stream=s)
        gpu.beam_gather(text, moved, 80, parents, rows=n, sources=n, status=status, stream=s)
        pool.reorder(old, then, parents, d[3], gain=3, workspace=more, stream=s)
        layers.copy(d[3], n, stream=s)

    buffers = [new, parents, tokens, moved, *d, d_refs, keys, values]

    def state():
        stream.synchronize()
        return [a.download(np.uint8, a.nbytes) for a in buffers]

    step(h)
    want = state()
    assert (d[3].download(np.int32, 3 * n) >= 0).any()
    graph = Graph(stream, lambda: step(h))
    for k in range(4):
        copy(d_refs, kept_refs, stream)
        for a in (new, parents, tokens, moved, d[1], d[2], d[3]):
            a.upload(np.full(a.nbytes // 4, 77, np.int32))
        if k % 2:
            gpu.beam_select(old_state, new_state, logits, vocab, parents, tokens,
                            workspace=space(work.nbytes))
            gpu.synchronize()
        graph.replay()
        for got, w in zip(state(), want):
            assert np.array_equal(got, w)
    gpu.check_status(status)
    graph.close(), stream.close()


def test_two_calls_at_once(gpu):
    """Two streams with workspaces of their own, and the same answers each time."""
    cases = [TreeCase("bf16", [900, 300], [60, 64], 2, 64, 16, 8, seed=k, max_length=9000).upload()
             for k in range(2)]
    want = [c.attention() for c in cases]
    streams = [Stream(), Stream()]
    for _ in range(5):
        for c in cases:
            c.out.upload(np.zeros(c.out.nbytes // 4, np.float32))
        for c, s in zip(cases, streams):
            c.case.paged.tree_attention(c.seqs, c.draft, c.d_query, c.out, 8, lse=c.lse,
                                        workspace=c.work, stream=s.handle)
        for s in streams:
            s.synchronize()
        for c, w in zip(cases, want):
            for got, x in zip(c.results(), w):
                assert np.array_equal(got, x)
    for s in streams:
        s.close()


def test_allocates_nothing(gpu):
    c = TreeCase("f16", [30, 5], [40, 3], 1, 64, 16, 4, seed=1, max_length=9000).upload()
    c.attention()
    parents, path = dev(np.concatenate(c.parents)), dev(np.zeros((2, 40)))
    draft = gpu.DraftTree(parents, c.d_mask, c.most, c.total, 2, starts=c.d_starts)
    tokens, counts = dev(np.zeros(c.total)), dev([0, 0])
    before = gpu.device_allocations()
    draft.build()
    c.case.paged.tree_attention(c.seqs, draft, c.d_query, c.out, 4, workspace=c.work)
    draft.accept(c.seqs, tokens, tokens, path, counts)
    gpu.PagedLayers([c.case.paged]).keep(c.seqs, path, 40, counts)
    gpu.synchronize()
    assert gpu.device_allocations() == before


def test_cpp_host_api(gpu):
    binary = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build",
                          "serving_api_test")
    r = subprocess.run([binary], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr
