"""Draft trees, page tables and beams on the host: what the operators over them
give, from their definitions, in whole numbers or 64 bits."""
import numpy as np

import nutllm_amd as nut
from paged_case import TYPES, Case, decode

U = 2.0 ** -24


def dev(a, dtype=np.int32):
    return nut.DeviceArray(like=np.asarray(a, dtype))


def space(need):
    """A workspace of `need` bytes that holds NaNs, or none."""
    a = nut.DeviceArray(like=np.full(max(need, 16), 0xff, np.uint8))
    a.nbytes = need
    return a


def words_of(sees):
    """Rows of truth values as mask words."""
    sees = np.asarray(sees, bool)
    pad = np.zeros((sees.shape[0], -(-sees.shape[1] // 32) * 32), bool)
    pad[:, :sees.shape[1]] = sees
    return (pad.reshape(len(sees), -1, 32).astype(np.uint64) <<
            np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)


def line_of(parents, i):
    got = []
    while i >= 0:
        got.append(i)
        i = parents[i]
    return got[::-1]


def tree_of(rng, m, shape="tree"):
    """Parents of m nodes: one root."""
    if shape == "chain":
        return [i - 1 for i in range(m)]
    if shape == "star":
        return [-1] + [0] * (m - 1) if m else []
    return [-1 if i == 0 else int(rng.integers(max(0, i // 3 - 1), i)) for i in range(m)]


def sees_of(parents):
    m = len(parents)
    sees = np.zeros((m, m), bool)
    for i in range(m):
        sees[i, line_of(parents, i)] = True
    return sees


def path_of(parents, tokens, chosen):
    path = [0] if len(parents) else []
    while path:
        after = [j for j in range(path[-1] + 1, len(parents))
                 if parents[j] == path[-1] and tokens[j] == chosen[path[-1]]]
        if not after:
            break
        path.append(after[0])
    return path


def attend64(q, k, v, scale):
    """(out, lse, bound of out's error, of lse's) of one query over rows k, v, as
    paged_case.Case derives them: a 16-bit row's products are dim times as many as
    limbs, whose sums add a 256th of the first one's roundings and a 65536th, under
    two for 256 components."""
    dim = len(q)
    q = np.asarray(q, np.float64)
    s = scale * (k @ q)
    p = np.exp(s - s.max())
    z = p.sum()
    ds = (dim + 6) * U * abs(scale) * (np.abs(k) @ np.abs(q)).max()
    rel = 2 * (ds + U * np.abs(s - s.max()).max() + 2 * U + (len(k) + 8) * U)
    lse = s.max() + np.log(z)
    return ((p / z) @ v, lse, rel * ((p / z) @ np.abs(v)) + 1e-30,
            rel + 2.0 ** -22 * (1 + abs(lse)))


class TreeCase:
    """Sequences of `held` rows with `counts` drafted nodes behind them, over a
    paged cache whose rows are all there; `lead` and `trail` node rows that no
    sequence names."""

    def __init__(self, kind, held, counts, kv, dim, page, heads, *, seed=0, sees=None,
                 slot_major=False, max_length=None, lead=0, trail=0, most=None, sigma=1.0,
                 stride=0):
        self.case = Case(kind, [n + m for n, m in zip(held, counts)], kv, dim, page, seed=seed,
                         slot_major=slot_major, max_length=max_length, sigma=sigma)
        self.held, self.counts, self.heads = list(held), list(counts), heads
        self.kind, self.kv, self.dim = kind, kv, dim
        rng = self.rng = np.random.default_rng(seed + 1000)
        self.starts = lead + np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.total, self.most = int(self.starts[-1]) + trail, most or max(1, max(counts))
        self.parents = [tree_of(rng, m) for m in counts]
        self.sees = [sees_of(p) for p in self.parents] if sees is None else sees
        self.stride = stride or -(-self.most // 32)
        self.mask = rng.integers(0, 1 << 32, (self.total, self.stride), np.uint64).astype(np.uint32)
        for b, s in enumerate(self.sees):
            if len(s):
                at = slice(self.starts[b], self.starts[b + 1])
                full = np.ones((len(s), self.stride * 32), bool)  # bits behind the nodes say nothing
                full[:, :len(s)] = s
                self.mask[at] = words_of(full)[:, :self.stride]
        self.query = (rng.standard_normal((self.total, heads, dim)) * 1.5).astype(np.float32)

    def upload(self, starts=True):
        self.case.upload()
        self.d_held = dev(self.held)
        self.d_mask, self.d_starts = dev(self.mask, np.uint32), dev(self.starts)
        self.d_query = dev(self.query, np.float32)
        self.status = self.case.d["status"]
        self.seqs = nut.PagedBatch(self.case.d["table"], self.case.width, self.d_held,
                                   len(self.held), self.case.max_length)
        self.draft = nut.DraftTree(None, self.d_mask, self.most, self.total, len(self.held),
                                   starts=self.d_starts if starts else None,
                                   mask_stride=self.stride, status=self.status)
        return self

    def attention(self, *, scale=None, stream=None, query=None, query_stride=0):
        """(out, lse) of the device; 7 where nothing was written."""
        self.out = dev(np.full((self.total, self.heads, self.dim), 7.0), np.float32)
        self.lse = dev(np.full((self.total, self.heads), 7.0), np.float32)
        self.work = space(self.case.paged.tree_attention_workspace(self.seqs, self.draft,
                                                                   self.heads))
        self.case.paged.tree_attention(self.seqs, self.draft, query or self.d_query, self.out,
                                       self.heads, scale=scale, lse=self.lse, stream=stream,
                                       query_stride=query_stride, workspace=self.work)
        nut.synchronize()
        return self.results()

    def results(self):
        n = self.total * self.heads
        return (self.out.download(np.float32, n * self.dim).reshape(self.total, self.heads, -1),
                self.lse.download(np.float32, n).reshape(self.total, self.heads))

    def expect(self, scale=None):
        """out, lse and bounds of their errors; 7 where nothing is written."""
        scale = self.dim ** -0.5 if scale is None else scale
        group = self.heads // self.kv
        out = np.full((self.total, self.heads, self.dim), 7.0)
        lse = np.full((self.total, self.heads), 7.0)
        tol, tol_lse = np.zeros_like(out), np.zeros_like(lse)
        for b, (n, m) in enumerate(zip(self.held, self.counts)):
            for h in range(self.heads if m else 0):
                k, v = (self.case.rows(p, b, h // group) for p in (self.case.keys,
                                                                   self.case.values))
                for i in range(m):
                    row = self.starts[b] + i
                    at = np.concatenate([np.arange(n), n + np.nonzero(self.sees[b][i])[0]])
                    if not len(at):
                        out[row, h], lse[row, h] = 0.0, -np.inf
                        continue
                    out[row, h], lse[row, h], tol[row, h], tol_lse[row, h] = attend64(
                        self.query[row, h], k[at], v[at], scale)
        return out, lse, tol, tol_lse

    def check(self, got=None, **kw):
        out, lse, tol, tol_lse = self.expect(kw.get("scale"))
        got, got_lse = got or self.attention(**kw)
        err = np.abs(got - out)
        assert np.all(err <= tol), (err / np.maximum(tol, 1e-30)).max()
        empty = np.isneginf(lse)
        assert np.array_equal(np.isneginf(got_lse), empty)
        assert np.all(np.abs(got_lse[~empty] - lse[~empty]) <= tol_lse[~empty])


# ------------------------------------------------------------------- pages --

class Pool:
    """A page pool with a table on the host and the device: rows of a table are
    -1 behind what a sequence holds."""

    def __init__(self, pages, page, batch, width, status=True):
        self.pages, self.page, self.batch, self.width = pages, page, batch, width
        self.refs = np.zeros(pages, np.int64)
        self.table = np.full((batch, width), -1, np.int64)
        self.lengths, self.held = np.zeros(batch, np.int64), np.zeros(batch, np.int64)
        self.status = dev([0])

    def reorder(self, parents, gains):
        """The definition: (table, lengths, held, copies), and the counts follow."""
        parents, gains = [int(p) for p in parents], [int(g) for g in gains]
        n = len(parents)
        table = np.full((n, self.width), -1, np.int64)
        lengths, held = np.zeros(n, np.int64), np.zeros(n, np.int64)
        copies = np.full((n, 3), -1, np.int64)
        free = [p for p in range(self.pages) if self.refs[p] == 0]
        before, seen = self.refs.copy(), set()
        for b in range(self.batch):
            for p in self.table[b, :self.held[b]]:
                if p >= 0:
                    self.refs[p] -= 1
        short = False
        for i, (p, gain) in enumerate(zip(parents, gains)):
            rows = int(self.lengths[p]) if p >= 0 else 0
            need, full = -(-(rows + gain) // self.page), rows // self.page
            for c in range(need):
                old = int(self.table[p, c]) if p >= 0 and c < self.held[p] else -1
                if c < full:
                    page = old
                elif p not in seen and old >= 0 and before[old] == 1:
                    page = old
                else:
                    page = free.pop(0) if free else -1
                    short = short or page < 0
                    if c == full and rows % self.page and page >= 0 and old >= 0:
                        copies[i] = old, page, rows % self.page
                table[i, c] = page
                if page >= 0:
                    self.refs[page] += 1
            lengths[i], held[i] = rows, need
            if p >= 0:
                seen.add(p)
        self.table, self.lengths, self.held, self.batch = table, lengths, held, n
        return copies, short

    def compact(self, limit, most):
        count = np.zeros(self.pages, np.int64)
        for b in range(self.batch):
            for p in self.table[b, :self.held[b]]:
                if p >= 0:
                    count[p] += 1
        high = [p for p in range(limit, self.pages)
                if self.refs[p] > 0 and self.refs[p] == count[p]]
        low = [p for p in range(limit) if self.refs[p] == 0]
        copies = np.full((most, 3), -1, np.int64)
        for k, (a, b) in enumerate(list(zip(high, low))[:most]):
            copies[k] = a, b, self.page
            self.refs[b], self.refs[a] = self.refs[a], 0
            for s in range(self.batch):
                row = self.table[s, :self.held[s]]
                row[row == a] = b
        return copies

    # device side
    def view(self):
        self.d_refs = dev(self.refs)
        return nut.PagePool(self.d_refs, self.pages, self.page, self.status)

    def place(self, table, lengths, held):
        d = [dev(table), dev(lengths), dev(held)]
        return d, nut.PageTable(d[0], self.width, d[1], d[2], len(lengths))


# ------------------------------------------------------------------- beams --

def beam_step(scores, lengths, ended, logits, keep, eos, power):
    """[requests][beams] states and logits [requests][beams][vocab] in 64 bits:
    (parents, tokens, scores, lengths, ended) and the ranks, best first."""
    requests, beams = scores.shape
    x = np.asarray(logits, np.float64)
    vocab = x.shape[-1]
    with np.errstate(all="ignore"):
        top = x.max(-1, keepdims=True)
        # the difference first: beside -1e30 a logarithm would be lost
        logp = (x - top) - np.log(np.exp(x - top).sum(-1, keepdims=True))
    got = [np.full((requests, keep), -1, np.int64), np.full((requests, keep), -1, np.int64),
           np.full((requests, keep), -np.inf), np.zeros((requests, keep), np.int64),
           np.zeros((requests, keep), np.int64)]
    ranks = np.full((requests, keep), -np.inf)
    for r in range(requests):
        found = []
        for i in range(beams):
            if not scores[r, i] > -np.inf:
                continue
            if ended is not None and ended[r, i]:
                n = 0 if lengths is None else int(lengths[r, i])
                found.append((float(scores[r, i]) / max(1, n) ** power, i, 0.0, eos,
                              float(scores[r, i]), n, 1))
                continue
            n = 1 + (0 if lengths is None else int(lengths[r, i]))
            total = float(scores[r, i]) + logp[r, i]
            best = np.lexsort((np.arange(vocab), -x[r, i]))[:keep]
            for v in best:
                if total[v] > -np.inf:
                    found.append((total[v] / max(1, n) ** power, i, x[r, i, v], int(v), total[v],
                                  n, int(ended is not None and v == eos)))
        found.sort(key=lambda f: (-f[0], f[1], -f[2], f[3]))
        for k, f in enumerate(found[:keep]):
            ranks[r, k] = f[0]
            got[0][r, k], got[1][r, k] = r * beams + f[1], f[3]
            got[2][r, k], got[3][r, k], got[4][r, k] = f[4], f[5], f[6]
    return got, ranks


__all__ = ["U", "TYPES", "Case", "Pool", "TreeCase", "attend64", "beam_step", "decode", "dev", "line_of",
           "path_of", "sees_of", "space", "tree_of", "words_of"]
