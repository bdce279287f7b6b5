"""Page tables of thousands of sequences, and caches of more layers than a launch takes."""
import numpy as np
import pytest

from paged_case import decode, encode, same
from serving_case import dev, space
from test_gpu_pages import Twin, _layers, _read

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("old,new", [(2048, 1024), (2049, 1025), (3001, 2500), (1, 2500),
                                     (2500, 1), (2048, 2049), (2049, 5000)])
def test_reorder_of_many_sequences(gpu, old, new):
    """Admissions, forks, growth and ends, with pages for all of it and without; more old
    sequences than shared memory counts, more new ones than the plan has threads."""
    rng = np.random.default_rng(old + new)
    t = Twin(gpu, 2 * old + 2 * new, 4, 1, 3)
    assert not t.reorder([-1] * old, gains=rng.integers(0, 9, old))
    t.grow(rng.integers(0, t.host.held * 4 + 1))
    parents = np.where(rng.random(new) < 0.2, -1, rng.integers(0, old, new))
    rows = np.where(parents < 0, 0, t.host.lengths[np.maximum(parents, 0)])
    t.reorder(parents, gains=np.minimum(rng.integers(0, 5, new), 12 - rows))
    t.reorder(np.arange(new), gain=0)
    t.reorder(rng.permutation(new)[:max(1, new // 2)], gain=0)
    # more than there are: the first ones get what is left
    n = t.host.batch
    parents = np.concatenate([np.arange(n), np.full(2 * old + 2 * new, -1)])
    assert t.reorder(parents, gains=np.where(parents < 0, 5, 0))


@pytest.mark.parametrize("parent", [0, 1500, 2999])
def test_reorder_forks_one_of_many(gpu, parent):
    """One sequence goes on 2,500 times, the others end."""
    t = Twin(gpu, 9000, 4, 1, 3)
    t.reorder([-1] * 3000, gains=[10 if b == parent else 2 for b in range(3000)])
    t.grow([10 if b == parent else 2 for b in range(3000)])
    t.reorder([parent] * 2500, gain=1)
    assert t.host.refs.max() == 2500
    t.reorder([2499, -1], gain=2)


@pytest.mark.parametrize("width,then", [(4, 9), (9, 4), (4, 1030)])
def test_reorder_to_another_width(gpu, width, then):
    """The new table's rows are longer, or shorter, than the old one's."""
    rng = np.random.default_rng(width)
    t = Twin(gpu, 4000, 4, 1, width)
    t.reorder([-1] * 9, gains=rng.integers(0, 17, 9))
    t.grow(rng.integers(0, t.host.held * 4 + 1))
    h = t.host
    parents, gains = np.array([3, 3, -1, 8, 0, 3]), np.array([0, 4, 16, 0, 3, 1])
    gains = np.where(parents < 0, gains, np.minimum(gains, 16 - h.lengths[np.maximum(parents, 0)]))
    if then > 1000:
        gains[2] = 4100
    old, h.width = t.now, then
    more = np.full((h.batch, max(0, then - width)), -1)
    h.table = np.concatenate([h.table, more], 1)[:, :max(then, width)]
    d, new = h.place(np.full((6, then), -1), np.full(6, -9), np.full(6, -9))
    copies = dev(np.full((6, 3), -9))
    t.pool.reorder(old, new, dev(parents), copies, gains=dev(gains),
                   workspace=space(t.pool.reorder_workspace(old, new)))
    want, short = h.reorder(parents, gains)
    assert not short and np.array_equal(copies.download(np.int32, 18).reshape(6, 3), want)
    t.d = d
    t.check()
    gpu.check_status(h.status)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("count,kv,page,dim,order", [(64, 1, 4, 16, "head"), (65, 2, 4, 16, "slot"),
                                                     (130, 1, 3, 40, "head")])
@pytest.mark.parametrize("bounds", [True, False])
def test_keep_in_many_layers(gpu, kind, count, kv, page, dim, order, bounds):
    rng, pages = np.random.default_rng(count), 11
    layers, hosts, status = _layers(gpu, kind, count, pages, kv, page, dim, order, rng, bounds)
    held, paths = [5, 2], [[0, 2, 3, 7], [1, 4]]
    table = rng.permutation(pages)[:10].reshape(2, 5)
    seqs = gpu.PagedBatch(dev(table), 5, dev(held), 2, 5 * page)
    gpu.PagedLayers(layers).keep(seqs, dev([p + [9] * (4 - len(p)) for p in paths]), 4,
                                 dev([len(p) for p in paths]))
    gpu.check_status(status)
    for host, got in _read(hosts, pages, kv, page, dim):
        for b, path in enumerate(paths):
            for k, i in enumerate(path):
                source, to = (table[b, (held[b] + x) // page] for x in (i, k))
                s, d = (held[b] + i) % page, (held[b] + k) % page
                if i == k:
                    continue
                for pool in host[:2]:
                    pool[to, :, d] = pool[source, :, s]
                if source != to and bounds:
                    row = decode(host[0][to, :, d], kind)
                    for e, f in ((0, np.minimum), (1, np.maximum)):
                        host[2][to, :, e] = encode(f(decode(host[2][to, :, e], kind), row), kind)
        assert all(same(a, b) for a, b in zip(got, host))


@pytest.mark.parametrize("kind,bits", [("f32", 0x7f800001), ("f32", 0xffc12345), ("f16", 0x7c01),
                                       ("f16", 0xfe55), ("bf16", 0x7f81), ("bf16", 0xffd5)])
@pytest.mark.parametrize("bounds", [True, False])
def test_keep_moves_bits(gpu, kind, bits, bounds):
    """Keys that are no numbers arrive as they were; the bounds of their page say so."""
    rng, pages, page = np.random.default_rng(3), 7, 4
    layers, hosts, status = _layers(gpu, kind, 2, pages, 2, page, 16, "head", rng, bounds)
    whole = np.uint32 if kind == "f32" else np.uint16
    for (host, flat, *_), pool in zip(hosts, (0, 1)):  # keys of one layer, values of the other
        host[pool].view(whole)[5, 1, 2, 3] = bits
        flat[pool].upload(host[pool])
    seqs = gpu.PagedBatch(dev([[2, 5, 1]]), 3, dev([3]), 1, 12)
    gpu.PagedLayers(layers).keep(seqs, dev([[3]]), 1, dev([1]))  # row 6, on page 5, to 3, on 2
    gpu.check_status(status)
    for i, (host, got) in enumerate(_read(hosts, pages, 2, page, 16)):
        for pool in host[:2]:
            pool[2, :, 3] = pool[5, :, 2]
        assert same(got[0], host[0]) and same(got[1], host[1])
        if bounds:
            none = np.isnan(decode(got[2], kind))
            assert none.sum() == (2 if i == 0 else 0) and np.all(none[2, 1, :, 3]) == (i == 0)
