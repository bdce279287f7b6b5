"""Draft trees over a paged KV cache against their definitions in 64 bits:
attention of every node, masks, accepted paths, the rows that stay. Slots that
no row occupies hold NaN, workspaces start as NaN, and bits of a mask behind a
sequence's nodes are set at random. Tolerances are derived in
serving_case.TreeCase.expect; whole numbers and moved rows are equal."""
import numpy as np
import pytest

import nutllm_amd as nut
from paged_case import decode, encode, same
from serving_case import TreeCase, attend64, dev, line_of, path_of, sees_of, tree_of, words_of

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,dim,page,slot_major", [
    (4, 2, 16, 16, False), (8, 2, 64, 16, False), (2, 2, 128, 32, True), (32, 4, 64, 64, False),
    (6, 2, 80, 24, True), (3, 1, 8, 1, False), (5, 1, 40, 7, False), (34, 2, 24, 128, True),
    (4, 1, 256, 16, False), (16, 1, 136, 5, True), (6, 6, 96, 16, False),
])
def test_attention(gpu, kind, heads, kv, dim, page, slot_major):
    held = [0, 1, 15, 16, 17, 31, 33, 64, 130, 0, 300, 47]
    counts = [1, 2, 3, 1, 17, 33, 5, 64, 8, 0, 20, 1]
    TreeCase(kind, held, counts, kv, dim, page, heads, seed=dim + page, slot_major=slot_major,
             lead=2, trail=3, stride=3).upload().check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("held,nodes", [(0, 1), (0, 33), (1, 64), (5, 65), (127, 100), (200, 257),
                                        (31, 1), (32, 32), (90, 129)])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 64), (8, 1, 64), (2, 2, 128), (3, 1, 32)])
def test_attention_sizes(gpu, kind, held, nodes, heads, kv, dim):
    """One sequence without starts: every block of query rows, masks of several words."""
    c = TreeCase(kind, [held], [nodes], kv, dim, 16, heads, seed=nodes + held)
    c.upload(starts=False).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", ["chain", "star"])
def test_attention_largest_tree(gpu, kind, shape):
    sees = [sees_of(tree_of(None, 1024, shape))]
    c = TreeCase(kind, [3], [1024], 1, 16, 32, 1, seed=4, sees=sees)
    c.upload().check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("held,counts,batch_dim", [([5000, 4097, 0, 1], [3, 70, 9, 2], 64),
                                                   ([9001], [40], 128), ([2047, 1025], [1, 1], 32)])
def test_attention_split_lengths(gpu, kind, held, counts, batch_dim):
    TreeCase(kind, held, counts, 1, batch_dim, 48, 4, seed=3).upload().check()


def test_attention_long(gpu):
    """Many runs, more than one piece of offsets each, a table wider than the sequence."""
    TreeCase("f16", [20011], [5], 1, 16, 64, 3, seed=5, max_length=33000).upload().check()
    TreeCase("bf16", [4100] * 40, [2] * 40, 8, 16, 16, 8, seed=6).upload().check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [8, 64, 80, 256])
@pytest.mark.parametrize("held,counts,heads", [([9000], [3], 2),
                                               ([8300, 40, 0, 6000], [64, 1, 0, 9], 4)])
def test_attention_many_parts(gpu, kind, dim, held, counts, heads):
    """Few query rows over long sequences, and some beside short ones: a row's parts are
    joined by several threads, which may have none of a short one."""
    TreeCase(kind, held, counts, 1, dim, 32, heads, seed=dim, max_length=12000).upload().check()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_any_mask(gpu, kind):
    """Masks that are no tree's: random ones, none, and nothing where no row is held."""
    rng = np.random.default_rng(1)
    counts, held = [40, 7, 33, 5], [0, 9, 31, 0]
    sees = [rng.random((m, m)) < 0.3 for m in counts]
    sees[0][5], sees[1][:] = False, False
    sees[3][:] = False
    TreeCase(kind, held, counts, 2, 64, 16, 8, seed=2, sees=sees).upload().check()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_is_that_of_one_token(gpu, kind):
    """A tree of one node reads what nut_paged_attention reads."""
    c = TreeCase(kind, [12, 300, 77], [1, 1, 1], 2, 64, 16, 8, seed=9).upload()
    got, lse = c.attention()
    one, one_lse = c.case.attention(c.query.reshape(3, 8, 64), 8)
    _, _, tol, tol_lse = c.expect()
    assert np.all(np.abs(got - one) <= 2 * tol) and np.all(np.abs(lse - one_lse) <= 2 * tol_lse)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads", [(64, 4), (80, 2), (128, 1), (256, 2)])
def test_unseen_rows_that_are_not_finite(gpu, kind, dim, heads):
    """Infinite and NaN keys and values in drafted rows: nodes that do not see them
    have their results as ever; those that see them do not have finite ones."""
    c = TreeCase(kind, [21, 0], [40, 9], 1, dim, 16, heads, seed=dim)
    bad = {0: [(3, "values", np.nan), (17, "values", np.inf), (18, "keys", np.nan),
               (30, "values", -np.inf), (39, "keys", np.inf)], 1: [(4, "values", np.nan)]}
    clean = c.expect()
    for b, rows in bad.items():
        for i, name, x in rows:
            row = c.held[b] + i
            p, slot = c.case.table[b, row // 16], row % 16
            getattr(c.case, name)[p, 0, slot] = encode(np.full(dim, x), kind)
    c.upload()
    got, lse = c.attention()
    out, want_lse, tol, tol_lse = clean
    for b, rows in bad.items():
        for i in range(c.counts[b]):
            at = c.starts[b] + i
            seen = {name for j, name, _ in rows if c.sees[b][i, j]}
            if not seen:
                assert np.all(np.abs(got[at] - out[at]) <= tol[at])
                assert np.all(np.abs(lse[at] - want_lse[at]) <= tol_lse[at])
            elif "values" in seen:
                assert not np.any(np.isfinite(got[at]))
                if seen == {"values"}:  # the weights are what they were
                    assert np.all(np.abs(lse[at] - want_lse[at]) <= tol_lse[at])


@pytest.mark.parametrize("kind", KINDS)
def test_values_that_are_not_finite_by_component(gpu, kind):
    """An infinite component that a node sees beside a NaN that it does not."""
    c = TreeCase(kind, [10], [6], 1, 64, 16, 2, seed=12,
                 sees=[sees_of([-1, 0, 0, 1, 1, 2])])
    p = c.case.table[0]
    for node, d, x in ((1, 3, np.inf), (2, 5, np.nan)):
        at = (p[(10 + node) // 16], 0, (10 + node) % 16, d)
        c.case.values[at] = encode(np.array([x]), kind)[0]
    out, _, tol, _ = TreeCase.expect(c)
    got, _ = c.upload().attention()
    sees = c.sees[0]
    for i in range(6):
        for d in range(64):
            if d == 3 and sees[i, 1]:
                assert np.all(got[i, :, d] == np.inf)
            elif d == 5 and sees[i, 2]:
                assert np.all(np.isnan(got[i, :, d]))
            elif d not in (3, 5):
                assert np.all(np.abs(got[i, :, d] - out[i, :, d]) <= tol[i, :, d])
            else:
                assert np.all(np.isfinite(got[i, :, d]))


@pytest.mark.parametrize("kind", KINDS)
def test_attention_large_and_small_values(gpu, kind):
    c = TreeCase(kind, [5, 77, 260], [3, 40, 18], 2, 32, 16, 4, seed=8, sigma=30.0)
    c.query *= 13.0
    c.upload().check()
    c.check(scale=0.0)
    c.check(scale=-0.25)


def test_attention_strided_queries(gpu):
    """Query rows with others' components between them; no log-sums asked for."""
    c = TreeCase("bf16", [50, 3], [9, 4], 2, 64, 16, 4, seed=3)
    wide = np.full((c.total, 4 * 64 + 20), np.nan, np.float32)
    wide[:, :256] = c.query.reshape(c.total, 256)
    c.upload().check(query=dev(wide, np.float32), query_stride=276)
    c.case.paged.tree_attention(c.seqs, c.draft, c.d_query, c.out, 4, workspace=c.work)
    out, _, tol, _ = c.expect()
    assert np.all(np.abs(c.results()[0] - out) <= tol)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", ["starts", "total", "most", "length", "longest", "page"])
def test_attention_of_what_it_cannot_follow(gpu, kind, bad):
    """The other sequences' results stand, and the check says what was wrong."""
    c = TreeCase(kind, [40, 20, 90], [6, 5, 7], 2, 64, 16, 4, seed=6, trail=4)
    c.upload()
    out, lse, tol, _ = c.expect()
    mine = slice(c.starts[1], c.starts[2])
    message = "rows out of range"
    left = None
    if bad == "starts":  # sequence 1 begins behind its end: 0 and 2 keep their nodes
        starts = c.starts.copy()
        starts[1] = starts[2] + 3
        c.d_starts.upload(starts)
        out[:], lse[:] = 7.0, 7.0
        # rows of sequence 0 now go up to 14, more than `most`
        out_2, _, tol_2, _ = c.expect()
        out[c.starts[2]:c.starts[3]] = out_2[c.starts[2]:c.starts[3]]
    elif bad == "total":
        starts = c.starts.copy()
        starts[3] = c.total + 1
        c.d_starts.upload(starts)
        out[c.starts[2]:] = 7.0
    elif bad == "most":
        c.draft.view.most = 6
        out[c.starts[2]:] = 7.0
    elif bad in ("length", "longest"):
        held = np.array(c.held, np.int32)
        held[1] = -1 if bad == "length" else c.case.max_length - 4
        c.d_held.upload(held)
        out[mine], lse[mine], message, left = 0.0, -np.inf, "length out of range", mine
    else:
        table = c.case.table.copy()
        table[1, 0] = c.case.pages
        c.case.d["table"].upload(table)
        message = "page out of range"
        out[mine] = np.nan
    got, got_lse = c.attention()
    there = ~np.isnan(out)
    assert np.all(np.abs(got - np.where(there, out, got))[there] <= tol[there])
    if left is not None:
        assert np.all(np.isneginf(got_lse[left]))
    if bad == "page":  # rows of the missing page have no part
        k0 = 16
        for h in range(4):
            k, v = (c.case.rows(p, 1, h // 2) for p in (c.case.keys, c.case.values))
            for i in range(5):
                at = np.concatenate([np.arange(k0, 20), 20 + np.nonzero(c.sees[1][i])[0]])
                row = c.starts[1] + i
                want, _, near, _ = attend64(c.query[row, h], k[at], v[at], 1 / 8)
                assert np.all(np.abs(got[row, h] - want) <= near)
    with pytest.raises(gpu.OutOfRange, match=message):
        gpu.check_status(c.status)
    gpu.check_status(c.status)


# ----------------------------------------------------------- mask, accept --

def _trees(seed=0):
    rng = np.random.default_rng(seed)
    counts = [1, 0, 2, 31, 32, 33, 64, 100, 5, 7]
    shapes = ["tree"] * 8 + ["chain", "star"]
    return rng, counts, [tree_of(rng, m, s) for m, s in zip(counts, shapes)]


@pytest.mark.parametrize("stride", [0, 6])
def test_mask(gpu, stride):
    rng, counts, parents = _trees()
    starts = 3 + np.concatenate([[0], np.cumsum(counts)])
    total, most = int(starts[-1]) + 2, max(counts)
    flat = np.full(total, -9, np.int32)
    want = np.full((total, stride or 4), 0xabcd1234, np.uint32)
    depth = np.full(total, 77, np.int32)
    for b, p in enumerate(parents):
        at = slice(starts[b], starts[b + 1])
        flat[at] = p
        if p:
            sees = np.zeros((len(p), 4 * 32), bool)
            sees[:, :len(p)] = sees_of(p)
            want[at, :4] = words_of(sees)
            depth[at] = [len(line_of(p, i)) - 1 for i in range(len(p))]
    mask, depths = dev(np.full(want.shape, 0xabcd1234), np.uint32), dev(np.full(total, 77))
    status = dev([0])
    draft = gpu.DraftTree(dev(flat), mask, most, total, len(counts), starts=dev(starts),
                          mask_stride=stride, status=status)
    draft.build(depths=depths)
    gpu.check_status(status)
    assert np.array_equal(mask.download(np.uint32, want.size).reshape(want.shape), want)
    assert np.array_equal(depths.download(np.int32, total), depth)


@pytest.mark.parametrize("shape", ["chain", "star", "tree"])
def test_mask_of_1024_nodes_without_starts(gpu, shape):
    rng = np.random.default_rng(3)
    parents = [tree_of(rng, 1024, shape) for _ in range(2)]
    mask = dev(np.zeros((2048, 32)), np.uint32)
    gpu.DraftTree(dev(np.concatenate(parents)), mask, 1024, 2048, 2).build()
    want = np.concatenate([words_of(sees_of(p)) for p in parents])
    assert np.array_equal(mask.download(np.uint32, want.size).reshape(want.shape), want)


@pytest.mark.parametrize("bad", [0, 5, -2, 1 << 30, -(1 << 31)])
def test_parents_that_are_none(gpu, bad):
    """A parent that is not below its node is taken for none, and reported."""
    parents = [-1, 0, 1, 1, 3, 2]
    flat = np.array(parents, np.int32)
    flat[3 if bad == 5 else 0 if bad == 0 else 4] = bad
    parents[3 if bad == 5 else 0 if bad == 0 else 4] = -1
    mask, status = dev(np.zeros((6, 1)), np.uint32), dev([0])
    draft = gpu.DraftTree(dev(flat), mask, 6, 6, 1, status=status)
    draft.build()
    with pytest.raises(gpu.OutOfRange, match="draft tree: parent out of range"):
        gpu.check_status(status)
    assert np.array_equal(mask.download(np.uint32, 6), words_of(sees_of(parents))[:, 0])
    path, counts = dev(np.full(6, -5)), dev([-5])
    seqs = gpu.PagedBatch(None, 0, dev([10]), 1, 100)
    tokens = dev(np.zeros(6))
    draft.accept(seqs, tokens, tokens, path, counts)
    with pytest.raises(gpu.OutOfRange, match="parent out of range"):
        gpu.check_status(status)
    want = path_of(parents, [0] * 6, [0] * 6)
    assert path.download(np.int32, len(want)).tolist() == want


@pytest.mark.parametrize("kinds", [1, 2, 3, 50])
def test_accept(gpu, kinds):
    """Paths of every length: with one token every node's lowest child is kept."""
    rng, counts, parents = _trees(kinds)
    starts = 2 + np.concatenate([[0], np.cumsum(counts)])
    total, most, batch = int(starts[-1]) + 1, 100, len(counts)
    tokens, chosen = rng.integers(0, kinds, (2, total))
    flat = np.full(total, -9, np.int32)
    for b, p in enumerate(parents):
        flat[starts[b]:starts[b + 1]] = p
    held = rng.integers(0, 500, batch)
    status = dev([0])
    draft = gpu.DraftTree(dev(flat), None, most, total, batch, starts=dev(starts), status=status)
    path, got, last, new = dev(np.full((batch, 104), -5)), dev([-5] * batch), dev([-5] * batch), \
        dev([-5] * batch)
    seqs = gpu.PagedBatch(None, 0, dev(held), batch, 700)
    draft.accept(seqs, dev(tokens), dev(chosen), path, got, path_stride=104, last=last,
                 new_lengths=new)
    gpu.check_status(status)
    path = path.download(np.int32, batch * 104).reshape(batch, 104)
    for b, p in enumerate(parents):
        at = slice(starts[b], starts[b + 1])
        want = path_of(p, tokens[at], chosen[at])
        assert path[b].tolist() == want + [-5] * (104 - len(want))
        assert got.download(np.int32, batch)[b] == len(want)
        assert new.download(np.int32, batch)[b] == held[b] + len(want)
        assert last.download(np.int32, batch)[b] == \
            (chosen[at][want[-1]] if want else -5)


def test_accept_of_what_does_not_fit(gpu):
    status = dev([0])
    draft = gpu.DraftTree(dev([-1, 0, -1, 0, -1, 0]), None, 2, 6, 3, status=status)
    path, counts, new = dev(np.full(6, -5)), dev([-5] * 3), dev([-5] * 3)
    draft.accept(gpu.PagedBatch(None, 0, dev([98, 99, -3]), 3, 100), dev([0] * 6), dev([0] * 6),
                 path, counts, new_lengths=new)
    assert counts.download(np.int32, 3).tolist() == [2, 0, 0]
    assert new.download(np.int32, 3).tolist() == [100, 99, -3]
    assert path.download(np.int32, 6).tolist() == [0, 1, -5, -5, -5, -5]
    with pytest.raises(gpu.OutOfRange, match="length out of range"):
        gpu.check_status(status)


# -------------------------------------------------------------------- keep --

def _host_keep(case, held, paths):
    for b, path in enumerate(paths):
        for k, i in enumerate(path):
            if i == k:
                continue
            source, to = (case.table[b, (held[b] + x) // case.page] for x in (i, k))
            s, t = (held[b] + i) % case.page, (held[b] + k) % case.page
            for pool in (case.keys, case.values):
                pool[to, :, t] = pool[source, :, s]
            if source != to:
                row = decode(case.keys[to, :, t], case.kind)
                for e, f in ((0, np.minimum), (1, np.maximum)):
                    case.bounds[to, :, e] = encode(
                        f(decode(case.bounds[to, :, e], case.kind), row), case.kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("kv,dim,page,slot_major", [(2, 16, 16, False), (4, 64, 16, True),
                                                    (1, 128, 7, False), (2, 80, 24, False),
                                                    (3, 8, 1, False), (1, 256, 64, False),
                                                    (2, 136, 5, True)])
@pytest.mark.parametrize("bounds", [True, False])
def test_keep(gpu, kind, kv, dim, page, slot_major, bounds):
    """Paths over one page and over many, in two layers at once."""
    held, counts = [0, 3, 15, 16, 40, 7, 30], [1, 9, 70, 20, 64, 0, 100]
    rng = np.random.default_rng(dim)
    paths = [sorted(rng.choice(m, min(m, rng.integers(1, 40)), replace=False).tolist())
             if m else [] for m in counts]
    paths[2] = list(range(70))  # all of it: nothing moves
    paths[4] = list(range(0, 64, 2))
    cases = [TreeCase(kind, held, counts, kv, dim, page, kv, seed=seed,
                      slot_major=slot_major).case.upload() for seed in (1, 1)]
    cases[1].keys[:], cases[1].values[:] = cases[0].values, cases[0].keys
    for b, n in enumerate(cases[1].lengths):
        for c in range(-(-int(n) // page)):
            p = cases[1].table[b, c]
            k = decode(cases[1].keys[p, :, :min(page, n - c * page)], kind)
            cases[1].bounds[p, :, 0] = encode(k.min(1), kind)
            cases[1].bounds[p, :, 1] = encode(k.max(1), kind)
    cases[1].upload()
    if not bounds:
        for c in cases:
            c.paged.view.d_bounds = None
    flat = np.full((len(paths), 101), 3, np.int32)
    for b, p in enumerate(paths):
        flat[b, :len(p)] = p
    seqs = gpu.PagedBatch(cases[0].d["table"], cases[0].width, dev(held), len(held),
                          cases[0].max_length)
    layers = gpu.PagedLayers([c.paged for c in cases])
    layers.keep(seqs, dev(flat), 101, dev([len(p) for p in paths]))
    cases[0].paged.check()
    for c in cases:
        before = c.bounds.copy()
        _host_keep(c, held, paths)
        for name in ("keys", "values"):
            assert same(c.pool(name), getattr(c, name))
        assert same(c.fetch("bounds"), c.bounds if bounds else before)


@pytest.mark.parametrize("bad,message", [("descends", "rows"), ("repeats", "rows"),
                                         ("negative", "rows"), ("far", "rows"),
                                         ("count", "rows"), ("negative count", "rows"),
                                         ("length", "length"), ("page", "page")])
def test_keep_of_what_it_cannot_follow(gpu, bad, message):
    """What stands before a bad entry is kept; other sequences are as ever."""
    held, counts = [20, 9], [30, 30]
    case = TreeCase("bf16", held, counts, 2, 64, 16, 2, seed=2).case.upload()
    path = [0, 2, 5, 9, 11, 12, 20, 21, 22, 23, 24, 25, 26, 27]
    flat, n, good = np.array([path, path], np.int32), [len(path)] * 2, list(path)
    d_held, table = list(held), case.table.copy()
    if bad in ("descends", "repeats", "negative", "far"):
        flat[0, 6] = {"descends": 3, "repeats": 12, "negative": -1, "far": 1 << 30}[bad]
        good = path[:6]
    elif bad == "count":
        n[0], good = 15, []
    elif bad == "negative count":
        n[0], good = -1, []
    elif bad == "length":
        d_held[0], good = case.max_length + 1, []
    else:  # rows 32 to 47 of sequence 0, nodes 12 to 27, are on a page that is not there
        table[0, 2] = -4
        case.d["table"].upload(table)
    seqs = gpu.PagedBatch(case.d["table"], case.width, dev(d_held), 2, case.max_length)
    gpu.PagedLayers([case.paged]).keep(seqs, dev(flat), 14, dev(n))
    with pytest.raises(gpu.OutOfRange, match=f"paged cache: {message} out of range"):
        case.paged.check()
    if bad == "page":
        good = [i if held[0] + i < 32 else k for k, i in enumerate(path)]
        good = [i if held[0] + k < 32 else k for k, i in enumerate(good)]
    _host_keep(case, held, [good, path])
    for name in ("keys", "values"):
        assert same(case.pool(name), getattr(case, name))
    assert same(case.fetch("bounds"), case.bounds)


def test_keep_far_into_a_large_pool(gpu):
    """Rows beyond 4 GiB of a pool: attention reads them, keep moves them."""
    pages, page, kv, dim = 40, 4096, 4, 128  # 4 MiB of bf16 a page and KV head row
    stride = 160 << 20  # bytes from page to page: 6.25 GiB
    keys, values = gpu.DeviceArray(nbytes=pages * stride), gpu.DeviceArray(nbytes=pages * stride)
    strides = (stride // 2, page * dim, dim)
    paged = gpu.PagedKV(keys, values, pages, page, kv, dim, gpu.BF16, strides=strides)
    rng = np.random.default_rng(0)
    n, m, where = page - 3, 6, [39, 2]
    k, v = (encode(rng.standard_normal((n + m, kv, dim)), "bf16") for _ in range(2))
    for array, rows in ((keys, k), (values, v)):
        for c, p in enumerate(where):
            for h in range(kv):
                part = np.ascontiguousarray(rows[c * page:(c + 1) * page, h])
                at = array.ptr.value + p * stride + h * page * dim * 2
                gpu.check(gpu.lib().nut_memcpy_h2d(at, part.ctypes.data, part.nbytes))
    q = rng.standard_normal((m, kv, dim)).astype(np.float32)
    seqs = gpu.PagedBatch(dev([where]), 2, dev([n]), 1, n + m)
    mask = dev(words_of(sees_of([-1, 0, 0, 1, 2, 2])), np.uint32)
    draft = gpu.DraftTree(None, mask, m, m, 1)
    out = dev(np.zeros((m, kv, dim)), np.float32)
    need = paged.tree_attention_workspace(seqs, draft, kv)
    work = gpu.DeviceArray(nbytes=need)
    paged.tree_attention(seqs, draft, dev(q, np.float32), out, kv, workspace=work)
    got = out.download(np.float32, q.size).reshape(q.shape)
    for i, parents in enumerate([[0], [0, 1], [0, 2], [0, 1, 3], [0, 2, 4], [0, 2, 5]]):
        at = list(range(n)) + [n + j for j in parents]
        for h in range(kv):
            want, _, near, _ = attend64(q[i, h], decode(k[at, h], "bf16"),
                                        decode(v[at, h], "bf16"), dim ** -0.5)
            assert np.all(np.abs(got[i, h] - want) <= near)
    gpu.PagedLayers([paged]).keep(seqs, dev([[0, 2, 5]]), 3, dev([3]))
    gpu.synchronize()
    for array, rows in ((keys, k), (values, v)):
        for to, of in ((n + 1, n + 2), (n + 2, n + 5)):
            for h in range(kv):
                row = np.empty(dim, np.uint16)
                at = array.ptr.value + where[to // page] * stride + (h * page + to % page) * dim * 2
                gpu.check(gpu.lib().nut_memcpy_d2h(row.ctypes.data, at, row.nbytes))
                assert np.array_equal(row, rows[of, h])
