"""A paged KV cache on the host, with its operators in 64 bits, and its copy
on the device."""
import numpy as np

import nutllm_amd as nut

TYPES = {"f32": nut.F32, "f16": nut.F16, "bf16": nut.BF16}


def encode(x, kind):
    """fp32 values as the cache's type stores them (to nearest, ties to even)."""
    x = np.asarray(x, np.float32)
    if kind == "f32":
        return x.copy()
    if kind == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = x.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def decode(a, kind):
    """float64 values of stored ones."""
    if kind != "bf16":
        return a.astype(np.float64)
    return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Case:
    """Sequences of the given lengths over pages in random order. Slots that no
    row occupies hold NaN. Host arrays are [pages][kv_heads][page][dim]."""

    def __init__(self, kind, lengths, kv_heads, dim, page, *, seed=0, slot_major=False,
                 max_length=None, spare=2, sigma=1.0, room=0):
        rng = self.rng = np.random.default_rng(seed)
        self.kind, self.kv, self.dim, self.page = kind, kv_heads, dim, page
        self.lengths = np.asarray(lengths, np.int32)
        self.batch = len(lengths)
        self.max_length = max_length or max(1, int(max(lengths)) + room)
        self.width = -(-self.max_length // page)
        self.pages = self.batch * self.width + spare
        order = rng.permutation(self.pages)[:self.batch * self.width]
        self.table = order.reshape(self.batch, self.width).astype(np.int32)
        self.slot_major = slot_major
        shape = (self.pages, kv_heads, page, dim)
        self.keys = encode(np.full(shape, np.nan), kind)
        self.values = self.keys.copy()
        for b, n in enumerate(self.lengths):
            for i in range(n):
                at = (self.table[b, i // page], slice(None), i % page)
                self.keys[at] = encode(rng.standard_normal((kv_heads, dim)) * sigma, kind)
                self.values[at] = encode(rng.standard_normal((kv_heads, dim)), kind)
        self.bounds = encode(np.full((self.pages, kv_heads, 2, dim), np.nan), kind)
        for b, n in enumerate(self.lengths):
            for c in range(-(-int(n) // page)):
                p = self.table[b, c]
                k = decode(self.keys[p, :, :min(page, n - c * page)], kind)
                self.bounds[p, :, 0] = encode(k.min(1), kind)
                self.bounds[p, :, 1] = encode(k.max(1), kind)
        self.weights = rng.random((self.batch, kv_heads, self.max_length)).astype(np.float32)
        self.positions = np.broadcast_to(np.arange(self.max_length, dtype=np.int32),
                                         self.weights.shape).copy()

    # ------------------------------------------------------------ device --

    def _lay(self, a):
        return np.ascontiguousarray(a.transpose(0, 2, 1, 3) if self.slot_major else a)

    def upload(self):
        A = nut.DeviceArray
        self.d = dict(keys=A(like=self._lay(self.keys)), values=A(like=self._lay(self.values)),
                      bounds=A(like=self.bounds), table=A(like=self.table),
                      lengths=A(like=self.lengths), weights=A(like=self.weights),
                      positions=A(like=self.positions), status=A(like=np.zeros(1, np.int32)),
                      new_lengths=A(like=np.full(self.batch, -7, np.int32)))
        strides = (self.page * self.kv * self.dim, self.dim, self.kv * self.dim)
        self.paged = nut.PagedKV(self.d["keys"], self.d["values"], self.pages, self.page, self.kv,
                                 self.dim, TYPES[self.kind],
                                 strides=strides if self.slot_major else None,
                                 bounds=self.d["bounds"], status=self.d["status"])
        self.seqs = nut.PagedBatch(self.d["table"], self.width, self.d["lengths"], self.batch,
                                   self.max_length)
        self.history = nut.PagedHistory(self.d["weights"], self.d["positions"], self.max_length)
        return self

    def pool(self, name):
        """The device's keys or values, as the host arrays lie."""
        host = getattr(self, name)
        a = self.d[name].download(host.dtype, host.size)
        if not self.slot_major:
            return a.reshape(host.shape)
        return a.reshape(self.pages, self.page, self.kv, self.dim).transpose(0, 2, 1, 3)

    def fetch(self, name):
        host = getattr(self, name)
        return self.d[name].download(host.dtype, host.size).reshape(host.shape)

    def new_lengths(self):
        return self.d["new_lengths"].download(np.int32, self.batch)

    def attention(self, query, heads, *, scale=None, history=None, selected=None, top=0,
                  stream=None, lse=True):
        """(out, lse) of the device."""
        dq = nut.DeviceArray(like=np.asarray(query, np.float32))
        out = nut.DeviceArray(like=np.full((self.batch, heads, self.dim), 7.0, np.float32))
        dl = nut.DeviceArray(like=np.full((self.batch, heads), 7.0, np.float32))
        ds = None if selected is None else nut.DeviceArray(like=np.asarray(selected, np.int32))
        need = self.paged.attention_workspace(self.seqs, heads, top=top,
                                              weighted=history is not None)
        work = nut.DeviceArray(like=np.full(max(1, need), 0xff, np.uint8))  # NaNs
        work.nbytes = need
        self.paged.attention(self.seqs, dq, out, heads, scale=scale, history=history, selected=ds,
                             top=top, lse=dl if lse else None, workspace=work, stream=stream)
        nut.synchronize()
        return (out.download(np.float32, self.batch * heads * self.dim)
                .reshape(self.batch, heads, self.dim),
                dl.download(np.float32, self.batch * heads).reshape(self.batch, heads))

    def select(self, query, heads, top, first, last):
        dq = nut.DeviceArray(like=np.asarray(query, np.float32))
        ds = nut.DeviceArray(like=np.full((self.batch, self.kv, top), -9, np.int32))
        need = self.paged.select_workspace(self.seqs, heads, top)
        work = nut.DeviceArray(like=np.full(need, 0xff, np.uint8))
        self.paged.select(self.seqs, dq, ds, heads, top, first=first, last=last, workspace=work)
        nut.synchronize()
        return ds.download(np.int32, self.batch * self.kv * top).reshape(self.batch, self.kv, top)

    def evict(self, budget, first=0, last=0):
        need = self.paged.evict_workspace(self.seqs, budget)
        work = nut.DeviceArray(like=np.full(need, 0xff, np.uint8))
        self.paged.evict(self.seqs, self.history, self.d["new_lengths"], budget, first=first,
                         last=last, workspace=work)
        nut.synchronize()

    # ---------------------------------------------------------- 64 bits --

    def rows(self, pool, b, h, n=None):
        n = int(self.lengths[b]) if n is None else n
        i = np.arange(n)
        return decode(pool[self.table[b, i // self.page], h, i % self.page], self.kind)

    def expect_attention(self, query, heads, scale=None, selected=None):
        """out, lse, the rows' weights summed over each group, and bounds of
        the error of out and of a row's weight (each relative to the weight).

        With u = 2^-24: a score is a sum of dim products, each rounded once
        and added with dim roundings at most, and the scaling of q and the
        conversion to base 2 add three more: |ds| <= (dim + 4) u sum |q k|.
        An exponential is off by 2 u and, through its argument, by |ds| and
        u |s - max|; the sums of n weights add n u relative at most, the join
        of runs 8 u more. Numerator and denominator both err."""
        scale = self.dim ** -0.5 if scale is None else scale
        group, u = heads // self.kv, 2.0 ** -24
        out = np.zeros((self.batch, heads, self.dim))
        lse = np.full((self.batch, heads), -np.inf)
        weights = np.zeros((self.batch, self.kv, self.max_length))
        tol_out, tol_w = np.zeros_like(out), np.zeros((self.batch, heads))
        q64 = np.asarray(query, np.float64)
        for b in range(self.batch):
            for h in range(heads):
                k, v = (self.rows(p, b, h // group) for p in (self.keys, self.values))
                if selected is not None:
                    at = np.concatenate([np.arange(c * self.page, min(len(k), (c + 1) * self.page))
                                         for c in selected[b, h // group] if c >= 0] or
                                        [np.zeros(0, int)])
                    k, v = k[at], v[at]
                if not len(k):
                    continue
                s = scale * (k @ q64[b, h])
                p = np.exp(s - s.max())
                z = p.sum()
                out[b, h], lse[b, h] = (p / z) @ v, s.max() + np.log(z)
                if selected is None:
                    weights[b, h // group, :len(k)] += p / z
                ds = (self.dim + 4) * u * scale * (np.abs(k) @ np.abs(q64[b, h])).max()
                rel = 2 * (ds + u * np.abs(s - s.max()).max() + 2 * u + (len(k) + 8) * u)
                tol_w[b, h] = rel
                tol_out[b, h] = rel * ((p / z) @ np.abs(v)) + 1e-30
        return out, lse, weights, tol_out, tol_w

    def expect_select(self, query, heads, top, first, last):
        got = np.full((self.batch, self.kv, top), -1, np.int32)
        group, q = heads // self.kv, np.asarray(query, np.float64)
        for b, n in enumerate(self.lengths):
            count = -(-int(n) // self.page)
            for h in range(self.kv):
                bound = decode(self.bounds[self.table[b, :count], h], self.kind)
                mine = q[b, h * group:(h + 1) * group, None]
                score = np.maximum(mine * bound[:, 0], mine * bound[:, 1]).sum(-1).max(0) \
                    if count else np.zeros(0)
                score[np.isnan(score)] = 1e300
                at = np.arange(count)
                score[(at < first) | (at >= count - last)] = np.inf
                best = np.sort(np.argsort(-score, kind="stable")[:top])
                got[b, h, :len(best)] = best
        return got

    def expect_evict(self, budget, first=0, last=0):
        """Evicts on the host arrays; the lengths that result."""
        for b, n in enumerate(self.lengths):
            n = int(n)
            if n <= budget:
                continue
            for h in range(self.kv):
                w = self.weights[b, h, :n].astype(np.float64)
                w[np.isnan(w)] = -np.inf
                pos = self.positions[b, h, :n].astype(np.int64)
                stay = (pos < first) | (pos > pos.max() - last)
                rank = sorted(range(n), key=lambda i: (not stay[i], 0 if stay[i] else -w[i], i))
                kept = np.zeros(n, bool)
                kept[rank[:budget]] = True
                holes, source = np.nonzero(~kept[:budget])[0], \
                    np.nonzero(kept[budget:])[0] + budget
                assert len(holes) == len(source)
                for i, j in zip(holes, source):
                    to, of = self.table[b, i // self.page], self.table[b, j // self.page]
                    for pool in (self.keys, self.values):
                        pool[to, h, i % self.page] = pool[of, h, j % self.page]
                    row = decode(self.keys[to, h, i % self.page], self.kind)
                    for e, f in ((0, np.minimum), (1, np.maximum)):
                        self.bounds[to, h, e] = encode(
                            f(decode(self.bounds[to, h, e], self.kind), row), self.kind)
                    for a in (self.weights, self.positions):
                        a[b, h, i] = a[b, h, j]
        return np.minimum(self.lengths, budget)

    def expect_append(self, keys, values, counts, history=True, firsts=None):
        """Appends fp32 rows [rows][kv][dim] on the host arrays."""
        row = 0
        for b, m in enumerate(counts):
            n = int(self.lengths[b])
            for j in range(m):
                i = n + j
                p, c = self.table[b, i // self.page], i % self.page
                self.keys[p, :, c] = encode(keys[row + j], self.kind)
                self.values[p, :, c] = encode(values[row + j], self.kind)
                new = decode(self.keys[p, :, c], self.kind)
                for e, f in ((0, np.minimum), (1, np.maximum)):
                    old = new if c == 0 else decode(self.bounds[p, :, e], self.kind)
                    self.bounds[p, :, e] = encode(f(old, new), self.kind)
                if history:
                    self.weights[b, :, i] = 0.0
                    self.positions[b, :, i] = (n if firsts is None else int(firsts[b])) + j
            row += m
        return self.lengths + np.asarray(counts, np.int32)


def same(a, b):
    """Equal bit for bit (NaN slots included)."""
    return np.array_equal(np.ascontiguousarray(a).view(np.uint8),
                          np.ascontiguousarray(b).view(np.uint8))
