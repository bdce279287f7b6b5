"""Page pools against their definition in whole numbers (serving_case.Pool):
tables that go from one step to the next, moves out of a cache's upper part, and
the copies that both ask for."""
import numpy as np
import pytest

import nutllm_amd as nut
from paged_case import TYPES, decode, encode, same
from serving_case import Pool, dev, space

pytestmark = pytest.mark.gpu


class Twin:
    """A pool on the host and on the device, stepped together. New tables start
    as -1, as the host's do, and copies as what no call writes."""

    def __init__(self, gpu, pages, page, batch, width):
        self.gpu, self.host = gpu, Pool(pages, page, batch, width)
        self.pool = self.host.view()
        self.d, self.now = self.host.place(self.host.table, self.host.lengths, self.host.held)

    def reorder(self, parents, gains=None, gain=0, stream=None):
        n, h = len(parents), self.host
        d, new = h.place(np.full((n, h.width), -1), np.full(n, -9), np.full(n, -9))
        copies = dev(np.full((n, 3), -9))
        work = space(self.pool.reorder_workspace(self.now, new))
        self.pool.reorder(self.now, new, dev(parents), copies,
                          gains=None if gains is None else dev(gains), gain=gain, workspace=work,
                          stream=stream)
        want, short = h.reorder(parents, [gain] * n if gains is None else gains)
        self.d, self.now, self.copies = d, new, copies
        assert np.array_equal(copies.download(np.int32, 3 * n).reshape(n, 3), want)
        self.check()
        if short:
            with pytest.raises(self.gpu.OutOfRange, match="page pool: out of pages"):
                self.gpu.check_status(h.status)
        self.gpu.check_status(h.status)
        return short

    def compact(self, limit, most):
        copies = dev(np.full((most, 3), -9))
        work = space(self.pool.compact_workspace(self.now))
        self.pool.compact(self.now, limit, copies, most, workspace=work)
        want = self.host.compact(limit, most)
        assert np.array_equal(copies.download(np.int32, 3 * most).reshape(most, 3), want)
        self.check()
        self.gpu.check_status(self.host.status)

    def check(self):
        h = self.host
        for got, want in zip(self.d, (h.table, h.lengths, h.held)):
            assert np.array_equal(got.download(np.int32, want.size).reshape(want.shape), want)
        assert np.array_equal(h.d_refs.download(np.int32, h.pages), h.refs)

    def grow(self, lengths):
        """Rows that an append put into pages that the sequences hold."""
        self.host.lengths[:] = lengths
        self.d[1].upload(self.host.lengths.astype(np.int32))


@pytest.mark.parametrize("pages,page,batch,width,seed", [
    (40, 4, 5, 9, 0), (300, 1, 12, 40, 1), (64, 16, 3, 70, 2), (5000, 8, 60, 33, 3),
    (9000, 3, 130, 200, 4), (33, 24, 1, 5, 5), (20000, 7, 40, 1100, 6),
])
def test_reorder_at_random(gpu, pages, page, batch, width, seed):
    """Sequences are admitted, grow, fork, give back and go, until pages run out too."""
    rng = np.random.default_rng(seed)
    t = Twin(gpu, pages, page, batch, width)
    shorts = 0
    for step in range(14):
        h = t.host
        n = int(rng.integers(1, 2 * batch + 1))
        kind = step % 4
        if kind == 0:  # admissions among sequences that go on
            parents = np.where(rng.random(n) < 0.5, -1, rng.integers(0, h.batch, n))
        elif kind == 1:  # every one goes on once
            parents, n = np.arange(h.batch), h.batch
        elif kind == 2:  # forks
            parents = rng.integers(0, h.batch, n)
        else:  # some go
            parents = rng.permutation(h.batch)[:max(1, h.batch // 2)]
            n = len(parents)
        rows = np.where(parents < 0, 0, h.lengths[np.maximum(parents, 0)])
        most = np.maximum(width * page - rows, 0)
        gains = np.minimum(rng.integers(0, page * max(2, width // 3), n), most)
        if step % 5 == 4:
            gain = int(min(3, most.min()))
            shorts += t.reorder(parents, gain=gain)
            gains = np.full(n, gain)
        else:
            shorts += t.reorder(parents, gains=gains)
        # append a part of what was reserved, but on pages that there are
        there = (t.host.table >= 0).cumprod(1).sum(1) * page
        t.grow(np.minimum(t.host.lengths + rng.integers(0, gains + 1),
                          np.maximum(there, t.host.lengths)))
        assert not np.any(t.host.refs < 0)
    print("steps without enough pages:", shorts)


def test_reorder_shares_and_parts(gpu):
    """Sequences of 10 rows, pages of 4: two full pages shared, the third parted."""
    t = Twin(gpu, 20, 4, 2, 6)
    t.reorder([-1, -1], gains=[10, 10])
    t.grow([10, 10])
    assert t.host.table[:, :3].tolist() == [[0, 1, 2], [3, 4, 5]]
    t.reorder([1, 0, 1, 1], gain=1)
    assert t.host.table[:, :3].tolist() == [[3, 4, 5], [0, 1, 2], [3, 4, 6], [3, 4, 7]]
    assert t.host.refs[:8].tolist() == [1, 1, 1, 3, 3, 1, 1, 1]
    t.reorder([2, 3], gain=8)  # the others go: their pages are free the next time
    assert t.host.refs[:8].tolist() == [0, 0, 0, 2, 2, 0, 1, 1]
    t.reorder([-1], gain=24)
    assert t.host.table[0].tolist() == [0, 1, 2, 5, 12, 13]  # 8 to 11 are freed with this call
    t.reorder([-1, -1], gain=0)
    assert not t.host.refs.any()


def test_reorder_pages_that_others_hold(gpu):
    """A partly filled page that something else holds too is parted, its holder's
    count stays; a prompt that another table keeps is shared."""
    t = Twin(gpu, 16, 4, 1, 5)
    t.reorder([-1], gain=10)
    t.grow([10])
    for page in (0, 2):
        t.host.refs[page] += 1
    t.host.d_refs.upload(t.host.refs.astype(np.int32))
    t.reorder([0], gain=2)
    assert t.host.table[0, :3].tolist() == [0, 1, 3]
    assert t.host.refs[:4].tolist() == [2, 1, 1, 1]


@pytest.mark.parametrize("bad", ["parent", "parent below", "length", "negative length", "held",
                                 "negative held", "gain", "negative gain", "page", "narrow"])
def test_reorder_of_what_it_cannot_follow(gpu, bad):
    t = Twin(gpu, 30, 4, 3, 6)
    t.reorder([-1, -1, -1], gains=[10, 9, 17])
    t.grow([10, 9, 17])
    h, parents, gains = t.host, np.array([1, 0, 2, 1]), np.array([1, 1, 1, 1])
    lengths, held, table = h.lengths.copy(), h.held.copy(), h.table.copy()
    before, old = h.refs.copy(), h.table.copy()
    message, empty, width = "length out of range", [0, 3], 6
    if bad in ("parent", "parent below"):
        parents[1] = 3 if bad == "parent" else -2
        message, empty = "parent out of range", [1]
    elif bad in ("length", "negative length"):
        lengths[1] = 13 if bad == "length" else -1
    elif bad in ("held", "negative held"):
        held[1] = 7 if bad == "held" else -1
    elif bad in ("gain", "negative gain"):
        gains[2] = 8 if bad == "gain" else -1
        message, empty = "rows out of range", []
    elif bad == "page":
        table[1, 0] = 30
        message, empty = "page out of range", []
    else:
        width, empty = 4, [2]  # 17 rows need five
    t.d[0].upload(table.astype(np.int32)), t.d[1].upload(lengths.astype(np.int32))
    t.d[2].upload(held.astype(np.int32))
    new = [dev(np.full((4, width), -1)), dev(np.full(4, -9)), dev(np.full(4, -9))]
    to = gpu.PageTable(new[0], width, new[1], new[2], 4)
    copies = dev(np.full((4, 3), -9))
    work = space(t.pool.reorder_workspace(t.now, to))
    t.pool.reorder(t.now, to, dev(parents), copies, gains=dev(gains), workspace=work)
    with pytest.raises(gpu.OutOfRange, match=message):
        gpu.check_status(h.status)
    gpu.check_status(h.status)
    got = new[0].download(np.int32, 4 * width).reshape(4, width)
    got_lengths, got_held = (a.download(np.int32, 4) for a in new[1:])
    refs = h.d_refs.download(np.int32, 30)
    assert refs.min() >= 0
    for i in range(4):
        rows = 0 if i in empty else int(h.lengths[parents[i]])
        gain = 0 if bad in ("gain", "negative gain") and i == 2 else 1
        need = -(-(rows + gain) // 4)
        if i in empty:
            assert got_lengths[i] == 0 and got_held[i] == 0 and np.all(got[i] == -1)
            continue
        assert got_lengths[i] == rows and got_held[i] == need
        full = old[parents[i], :rows // 4].copy()
        if bad == "page" and parents[i] == 1:
            full[0] = -1
        assert got[i, :rows // 4].tolist() == full.tolist()
        assert np.all(got[i, rows // 4:need] >= 0) and np.all(got[i, need:] == -1)
    # the counts are those of the entries, and of what nobody could give back
    count = np.zeros(30, int)
    np.add.at(count, got[got >= 0], 1)
    lost = old[1, :h.held[1]] if bad in ("held", "negative held") else \
        old[1, :1] if bad == "page" else []
    for p in lost:
        count[p] += 1
    assert refs.tolist() == count.tolist(), (refs - count, before)


def test_reorder_large_pool(gpu):
    """Two million pages: several spans a segment, free ones here and there."""
    pages = 2_000_003
    rng = np.random.default_rng(0)
    t = Twin(gpu, pages, 16, 1, 50)
    free = np.sort(rng.choice(pages, 40, replace=False))
    t.host.refs[:] = 1
    t.host.refs[free] = 0
    t.host.d_refs.upload(t.host.refs.astype(np.int32))
    n = [dev(np.full((2, 50), -1)), dev([-9] * 2), dev([-9] * 2)]
    to = gpu.PageTable(n[0], 50, n[1], n[2], 2)
    work = space(t.pool.reorder_workspace(t.now, to))
    t.pool.reorder(t.now, to, dev([-1, -1]), dev(np.zeros((2, 3))), gains=dev([240, 400]),
                   workspace=work)
    gpu.check_status(t.host.status)
    got = n[0].download(np.int32, 100).reshape(2, 50)
    assert got[0, :15].tolist() == free[:15].tolist()
    assert got[1, :25].tolist() == free[15:].tolist()
    assert t.host.d_refs.download(np.int32, pages).min() == 1


@pytest.mark.parametrize("pages,page,batch,width,seed", [(64, 16, 3, 9, 0), (500, 4, 17, 30, 1),
                                                         (9001, 8, 90, 60, 2), (20, 1, 2, 9, 3)])
def test_compact_at_random(gpu, pages, page, batch, width, seed):
    rng = np.random.default_rng(seed)
    t = Twin(gpu, pages, page, batch, width)
    t.reorder([-1] * batch, gains=rng.integers(0, width * page // 2, batch))
    t.grow(rng.integers(0, t.host.held * page + 1))
    t.reorder(rng.integers(0, batch, batch), gain=1)
    t.reorder(rng.permutation(batch)[:(batch + 1) // 2], gain=0)
    used = np.nonzero(t.host.refs)[0]
    if len(used):
        t.host.refs[used[-1]] += 1  # something else holds it: it stays
        t.host.d_refs.upload(t.host.refs.astype(np.int32))
    for limit, most in ((pages // 2, 3), (pages // 3, 2 * pages), (pages, 1), (0, 5),
                        (max(1, len(used)), pages)):
        t.compact(limit, most)


@pytest.mark.parametrize("pages,batch,width,most", [(4096, 90, 60, 4096), (4097, 90, 60, 700),
                                                    (300, 17, 4000, 300), (300, 17, 30, 70000),
                                                    (4096, 1, 16384, 16384), (4096, 1, 16385, 9),
                                                    (500, 128, 9, 50), (500, 129, 9, 50),
                                                    (700, 5, 90, 16385), (1, 1, 1, 1)])
def test_compact_by_one_workgroup_or_more(gpu, pages, batch, width, most):
    """Pools, tables and lists at the sizes where one workgroup follows them all, and behind."""
    rng = np.random.default_rng(pages + width)
    t = Twin(gpu, pages, 2, batch, width)
    gains = rng.integers(0, min(width * 2, 2 * pages // batch) + 1, batch)
    t.reorder([-1] * batch, gains=gains)
    t.grow(rng.integers(0, t.host.held * 2 + 1))
    t.reorder(rng.integers(0, batch, batch), gain=1)
    t.compact(pages // 2, most)
    t.compact(pages // 3, most)


def test_compact_missing_pages(gpu):
    t = Twin(gpu, 12, 4, 2, 4)
    t.reorder([-1, -1], gain=12)
    t.reorder([1], gain=12)
    t.host.table[0, 1] = 99
    t.d[0].upload(t.host.table.astype(np.int32))
    copies = dev(np.full((4, 3), -9))
    t.pool.compact(t.now, 3, copies, 4, workspace=space(t.pool.compact_workspace(t.now)))
    with pytest.raises(gpu.OutOfRange, match="page out of range"):
        gpu.check_status(t.host.status)
    assert t.d[0].download(np.int32, 4).tolist() == [0, 99, 1, -1]
    assert copies.download(np.int32, 12).reshape(4, 3).tolist() == \
        [[3, 0, 4], [5, 1, 4], [-1] * 3, [-1] * 3]
    t.d[2].upload(np.array([5], np.int32))
    t.pool.compact(t.now, 3, copies, 4, workspace=space(t.pool.compact_workspace(t.now)))
    with pytest.raises(gpu.OutOfRange, match="length out of range"):
        gpu.check_status(t.host.status)


# -------------------------------------------------------------------- copy --

def _layers(gpu, kind, count, pages, kv, page, dim, order, rng, bounds=True):
    """Views and host arrays [pages][kv][page][dim] of `count` layers; pages, slots
    or heads first, with room between the rows of one layout."""
    layers, hosts, status = [], [], dev([0])
    for _ in range(count):
        host = [encode(rng.standard_normal((pages, kv, page, dim)), kind) for _ in range(2)]
        host.append(encode(rng.standard_normal((pages, kv, 2, dim)), kind))
        row = dim + (16 if order == "room" else 0)
        strides = {"head": (kv * page * row, page * row, row), "room": (kv * page * row,
                                                                      page * row, row),
                   "slot": (kv * page * row, row, kv * row),
                   "heads first": (page * row, pages * page * row, row)}[order]
        flat = []
        for a in host[:2]:
            wide = np.zeros((pages, kv, page, row), a.dtype)
            wide[..., :dim] = a
            axes = {"slot": (0, 2, 1, 3), "heads first": (1, 0, 2, 3)}.get(order, (0, 1, 2, 3))
            flat.append(nut.DeviceArray(like=np.ascontiguousarray(wide.transpose(axes))))
        b = nut.DeviceArray(like=host[2])
        layers.append(gpu.PagedKV(*flat, pages, page, kv, dim, TYPES[kind], strides=strides,
                                  bounds=b if bounds else None, status=status))
        hosts.append((host, flat, b, axes, row))
    return layers, hosts, status


def _read(hosts, pages, kv, page, dim):
    for host, flat, b, axes, row in hosts:
        shape = [(pages, kv, page, row)[a] for a in axes]
        back = np.argsort(axes)
        got = [f.download(h.dtype, int(np.prod(shape))).reshape(shape).transpose(back)[..., :dim]
               for f, h in zip(flat, host)]
        yield host, got + [b.download(host[2].dtype, host[2].size).reshape(host[2].shape)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("count,kv,page,dim,order", [
    (1, 2, 16, 64, "head"), (3, 3, 24, 80, "slot"), (66, 1, 4, 16, "head"), (2, 4, 64, 128, "room"),
    (2, 1, 1, 8, "slot"), (2, 2, 5, 256, "heads first"), (2, 5, 300, 40, "head"),
])
@pytest.mark.parametrize("bounds", [True, False])
def test_copy(gpu, kind, count, kv, page, dim, order, bounds):
    """Whole pages and parts of them, none and empty ones, in every layer."""
    rng, pages = np.random.default_rng(dim + page), 11
    layers, hosts, status = _layers(gpu, kind, count, pages, kv, page, dim, order, rng, bounds)
    copies = [[3, 7, page], [3, 0, page // 2], [-1, -1, -1], [10, 2, 1], [5, 5, page],
              [4, 6, 0], [-7, 99, 99]]
    gpu.PagedLayers(layers).copy(dev(copies), len(copies))
    gpu.check_status(status)
    for host, got in _read(hosts, pages, kv, page, dim):
        for a, b, rows in copies:
            if a < 0:
                continue
            for pool in host[:2]:
                pool[b, :, :rows] = pool[a, :, :rows]
            if bounds:
                host[2][b] = host[2][a]
        for a, b in zip(got, host):
            assert same(a, b)


@pytest.mark.parametrize("entry,message", [([11, 2, 4], "page"), ([3, 11, 4], "page"),
                                           ([3, -1, 4], "page"), ([3, 2, 5], "rows"),
                                           ([3, 2, -1], "rows")])
def test_copy_of_what_it_cannot_follow(gpu, entry, message):
    rng = np.random.default_rng(0)
    layers, hosts, status = _layers(gpu, "f16", 2, 11, 2, 4, 16, "head", rng)
    gpu.PagedLayers(layers).copy(dev([entry, [1, 9, 4]]), 2)
    with pytest.raises(gpu.OutOfRange, match=f"{message} out of range"):
        gpu.check_status(status)
    for host, got in _read(hosts, 11, 2, 4, 16):
        for a in host:
            a[9] = a[1]
        assert all(same(a, b) for a, b in zip(got, host))


def test_copy_of_nothing(gpu):
    rng = np.random.default_rng(0)
    layers, hosts, status = _layers(gpu, "f16", 1, 3, 1, 4, 16, "head", rng)
    gpu.PagedLayers(layers).copy(None, 0)
    gpu.check_status(status)


def test_beams_over_pages(gpu):
    """What forked sequences hold is what they held, row by row, through steps of
    a reorder, its copies and an append: in two layers, with bounds."""
    kind, kv, dim, page, pages, width = "bf16", 2, 16, 4, 64, 12
    rng = np.random.default_rng(5)
    layers, hosts, status = _layers(gpu, kind, 2, pages, kv, page, dim, "head", rng)
    cache, t = gpu.PagedLayers(layers), Twin(gpu, pages, page, 1, width)
    texts = [np.zeros((0, 2, 2, kv, dim), np.float32)]
    parents, gain = [-1, -1], 5
    for step in range(24):
        texts = [texts[p] if p >= 0 else np.zeros((0, 2, 2, kv, dim), np.float32) for p in parents]
        t.reorder(parents, gain=gain)
        cache.copy(t.copies, len(parents))
        new = rng.standard_normal((len(parents), gain, 2, 2, kv, dim)).astype(np.float32)
        starts = dev(np.arange(len(parents) + 1) * gain)
        seqs = gpu.PagedBatch(t.d[0], width, t.d[1], len(parents), width * page)
        grown = dev(np.zeros(len(parents)))
        for l, view in enumerate(layers):
            k, v = (dev(new[:, :, l, i].reshape(-1, kv, dim), np.float32) for i in range(2))
            view.append(seqs, k, v, grown, starts=starts, max_new=gain)
        texts = [np.concatenate([x, n]) for x, n in zip(texts, new)]
        t.grow(t.host.lengths + gain)
        assert grown.download(np.int32, len(parents)).tolist() == t.host.lengths.tolist()
        for l, (_, got) in enumerate(_read(hosts, pages, kv, page, dim)):
            for b, text in enumerate(texts):
                at = np.arange(len(text))
                p, slot = t.host.table[b][at // page], at % page
                for i in range(2):
                    assert same(got[i][p, :, slot], encode(text[:, l, i], kind))
                for c in range(-(-len(text) // page)):
                    k = decode(encode(text[c * page:(c + 1) * page, l, 0], kind), kind)
                    bound = decode(got[2][t.host.table[b, c]], kind)
                    # a copied page's bounds cover what its source had, and no less
                    assert np.all(bound[:, 0] <= k.min(0)) and np.all(bound[:, 1] >= k.max(0))
        n = len(parents)
        parents = rng.integers(0, n, int(rng.integers(2, 7))).tolist()
        if len(texts[0]) > 30:
            parents = [-1, -1]
        gain = int(rng.integers(1, 4))
    gpu.check_status(status)
