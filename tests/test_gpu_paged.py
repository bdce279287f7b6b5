"""The paged KV cache's operators against their definitions in 64 bits: sizes
at the edges of pages and tiles, empty sequences, every type and layout, NaN in
the slots behind a sequence's end, workspaces that start as NaN. Tolerances are
derived in paged_case.Case.expect_attention; what is moved or chosen is
compared bit for bit."""
import numpy as np
import pytest

from paged_case import Case, decode, encode, same

pytestmark = pytest.mark.gpu

EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300]


def query_of(case, heads, seed=1, sigma=1.5):
    rng = np.random.default_rng(seed)
    return (rng.standard_normal((case.batch, heads, case.dim)) * sigma).astype(np.float32)


def check_attention(case, heads, query, **kw):
    out, lse, weights, tol, tol_w = case.expect_attention(query, heads,
                                                          selected=kw.get("selected"))
    got, got_lse = case.attention(query, heads, **kw)
    err = np.abs(got - out) / np.where(tol > 0, tol, 1)
    print(f"worst error {err.max():.3f} of its bound", flush=True)
    assert np.all(np.abs(got - out) <= tol)
    empty = np.isneginf(lse)
    assert np.array_equal(np.isneginf(got_lse), empty)
    # the logarithm's argument errs as a weight does, and its result is rounded
    assert np.all(np.abs(got_lse[~empty] - lse[~empty]) <=
                  (tol_w + 2.0 ** -22 * (1 + np.abs(lse)))[~empty])
    return weights, tol_w


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim,page,slot_major", [
    (4, 2, 16, 16, False), (8, 2, 64, 16, False), (2, 2, 128, 32, True), (32, 4, 64, 64, False),
    (6, 2, 80, 24, True), (3, 1, 8, 1, False), (5, 1, 40, 7, False), (34, 2, 24, 128, True),
    (4, 1, 256, 16, False), (16, 1, 136, 5, True),
])
def test_attention(gpu, kind, heads, kv, dim, page, slot_major):
    case = Case(kind, EDGES, kv, dim, page, seed=dim + page, slot_major=slot_major).upload()
    check_attention(case, heads, query_of(case, heads))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 16), (3, 1, 40), (8, 8, 64), (34, 2, 96),
                                          (2, 2, 128), (5, 1, 136), (4, 2, 256)])
@pytest.mark.parametrize("most", [1, 3, 16, 17, 32, 33, 48, 64, 65])
def test_attention_short(gpu, kind, heads, kv, dim, most):
    """Sequences of one tile, two and more: with weights, and of a selection."""
    lengths = [most, 0, 1, max(1, most - 1), most // 2]
    case = Case(kind, lengths, kv, dim, 8, seed=most, max_length=most).upload()
    q = query_of(case, heads)
    check_attention(case, heads, q)
    check_attention(case, heads, q, history=case.history)
    pages = (most + 7) // 8
    top = min(pages, 4)
    selected = np.full((5, kv, top), -1, np.int32)
    for b, n in enumerate(lengths):
        for h in range(kv):
            there = case.rng.permutation((n + 7) // 8)[:top]
            selected[b, h, :len(there)] = there
    check_attention(case, heads, q, selected=selected, top=top)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lengths", [[1500], [2049, 1, 0, 1024, 1023, 1025], [5000, 4097]])
def test_attention_split_lengths(gpu, kind, lengths):
    case = Case(kind, lengths, 1, 64, 48, seed=3).upload()
    check_attention(case, 4, query_of(case, 4, sigma=3.0))


def test_attention_long(gpu):
    """A length that many runs share, with a table wider than the sequence."""
    case = Case("f16", [20011], 1, 16, 64, seed=5, max_length=33000).upload()
    check_attention(case, 3, query_of(case, 3))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_attention_large_and_small_values(gpu, kind):
    """Scores of hundreds either way, a row that takes all the weight, queries
    far from one; without the log-sum-exp."""
    case = Case(kind, [5, 77, 260], 2, 32, 16, seed=8, sigma=30.0)
    case.upload()
    q = query_of(case, 4, sigma=20.0)
    out, _, _, tol, _ = case.expect_attention(q, 4)
    got, lse = case.attention(q, 4, lse=False)
    assert np.all(np.abs(got - out) <= tol) and np.all(lse == 7.0)
    for power in (-60, 40):
        q = query_of(case, 4) * np.float32(2.0 ** power)
        scale = float(2.0 ** -power / 8)
        out, _, _, tol, _ = case.expect_attention(q, 4, scale=scale)
        got, _ = case.attention(q, 4, scale=scale)
        assert np.all(np.abs(got - out) <= tol)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("power", [0, 10, 16, 20, 25, 40])
def test_attention_one_large_query_component(gpu, kind, power):
    """A component 2^power above the others that the rows do not have, or have
    in part. An fp16 row's query component is held to 2^-23 of itself and 2^-38
    of the largest one, its weight to 2^-23 and 2^-39 of the largest: a score
    errs by scale sum (2^-23 |q_d| + 2^-38 max |q|) |k_d| more, and a result,
    whose largest weight is 1 before the division by z >= 1, by
    sum (2^-23 p + 2^-39) |v| / z."""
    case = Case(kind, [30, 250], 2, 64, 16, seed=87)
    rows = decode(case.keys, kind)
    rows[..., 11] = 0.0
    rows[case.table[1], 1, :, 11] = 2.0 ** -min(power, 14)
    case.keys[:] = encode(rows, kind)
    case.upload()
    q = query_of(case, 4)
    q[..., 11] = np.float32(2.0 ** power)
    out, _, _, tol, _ = case.expect_attention(q, 4)
    if kind == "f16":
        for b, n in enumerate(case.lengths):
            for h in range(4):
                k, v = (np.abs(case.rows(p, b, h // 2)) for p in (case.keys, case.values))
                size = np.abs(q[b, h].astype(np.float64))
                ds = (k @ (2.0 ** -23 * size + 2.0 ** -38 * size.max())).max() / 8
                # both parts of the quotient err by ds of each weight
                tol[b, h] += (2 * ds + 2.0 ** -23 + n * 2.0 ** -39) * v.max(0)
    got, _ = case.attention(q, 4)
    print(f"worst error {(np.abs(got - out) / tol).max():.3f} of its bound", flush=True)
    assert np.all(np.abs(got - out) <= tol)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_attention_infinite_keys(gpu, kind):
    """Rows whose score is minus infinity weigh nothing, a sequence of such
    rows alone gives zeros; a NaN key shows in its own KV head only."""
    case = Case(kind, [40, 3, 33], 2, 32, 16, seed=9)
    q = np.abs(query_of(case, 4)) + np.float32(0.1)
    inf = encode(np.array(-np.inf), kind)
    plain = Case(kind, [40, 3, 33], 2, 32, 16, seed=9)
    for i in (0, 17, 39):  # sequence 0: these rows
        case.keys[case.table[0, i // 16], :, i % 16, 5] = inf
    for i in range(3):     # sequence 1: all rows
        case.keys[case.table[1, 0], :, i, 5] = inf
    case.keys[case.table[2, 1], 1, 3, 0] = encode(np.array(np.nan), kind)
    case.upload()
    got, lse = case.attention(q, 4)
    assert np.all(got[1] == 0) and np.all(np.isneginf(lse[1]))
    assert np.all(np.isnan(got[2, 2:])) and np.all(np.isfinite(got[2, :2]))
    keep = [i for i in range(40) if i not in (0, 17, 39)]
    for h in range(4):
        k, v = (plain.rows(p, 0, h // 2)[keep] for p in (plain.keys, plain.values))
        s = k @ q[0, h].astype(np.float64) * 32 ** -0.5
        p = np.exp(s - s.max())
        want, size = (p / p.sum()) @ v, (p / p.sum()) @ np.abs(v)
        _, _, _, _, tol_w = plain.expect_attention(q, 4)
        assert np.all(np.abs(got[0, h] - want) <= tol_w[0, h] * size)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [32, 128])
@pytest.mark.parametrize("length", [1, 20, 40, 100, 2500])
def test_attention_of_no_weight_over_odd_values(gpu, kind, dim, length):
    """A head whose scores are all minus infinity gets zeros and minus infinity
    whatever its rows' values are, in one run and in several, and its rows no
    weight; the other KV head gets what it would."""
    case = Case(kind, [length, 33], 2, dim, 16, seed=83)
    q = np.abs(query_of(case, 4)) + np.float32(0.1)
    out, _, weights, tol, tol_w = case.expect_attention(q, 4)
    for i in range(length):
        at = (case.table[0, i // 16], 1, i % 16)
        case.keys[at][3] = encode(np.array(-np.inf), kind)
        case.values[at][i % dim] = encode(np.array((np.inf, -np.inf, np.nan)[i % 3]), kind)
    before = case.weights.copy()
    case.upload()
    for history in (None, case.history):
        got, lse = case.attention(q, 4, history=history)
        assert np.all(got[0, 2:] == 0) and np.all(np.isneginf(lse[0, 2:]))
        assert np.all(np.abs(got - out)[0, :2] <= tol[0, :2])
        assert np.all(np.abs(got - out)[1] <= tol[1])
    grown = case.fetch("weights") - before
    assert np.all(grown[0, 1] == 0)
    assert np.all(np.abs(grown - weights)[0, 0, :length] <=
                  weights[0, 0, :length] * tol_w[0, :2].max() + 2.0 ** -22)
    pages = np.arange(-(-length // 16))
    chosen = np.full((2, 2, max(3, len(pages))), -1, np.int32)
    chosen[0, :, :len(pages)], chosen[1] = pages, np.r_[0:3, [-1] * (chosen.shape[2] - 3)]
    got, lse = case.attention(q, 4, selected=chosen, top=chosen.shape[2])
    assert np.all(got[0, 2:] == 0) and np.all(np.isneginf(lse[0, 2:]))
    assert np.all(np.abs(got - out)[0, :2] <= tol[0, :2])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 64, 16), (3, 3, 128, 32), (34, 2, 24, 9)])
def test_attention_gathers_weights(gpu, kind, heads, kv, dim, page):
    lengths = [0, 1, 33, 128, 700, 1300]
    case = Case(kind, lengths, kv, dim, page, seed=11).upload()
    before = case.weights.copy()
    q = query_of(case, heads)
    weights, tol_w = check_attention(case, heads, q, history=case.history)
    case.attention(q, heads, history=case.history, lse=False)  # a second token
    got = case.fetch("weights").astype(np.float64)
    group = heads // kv
    for b, n in enumerate(lengths):
        rel = tol_w[b].reshape(kv, group).max(1)[:, None]
        # two additions to the weight that was there, each rounded once
        want = before[b] + 2 * weights[b]
        bound = 2 * weights[b] * (rel + group * 2.0 ** -24) + 2 * 2.0 ** -24 * want + 1e-37
        assert np.all(np.abs(got[b] - want) <= bound)
        assert same(case.fetch("weights")[b, :, n:], before[b, :, n:])
    assert same(case.fetch("positions"), case.positions)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim,page,top,first,last", [
    (8, 2, 64, 16, 8, 1, 2), (2, 2, 128, 8, 5, 0, 0), (32, 4, 64, 4, 31, 1, 1),
    (6, 2, 80, 24, 4, 0, 1), (34, 2, 24, 3, 16, 16, 0), (4, 1, 256, 16, 1, 0, 1),
])
def test_select_and_sparse_attention(gpu, kind, heads, kv, dim, page, top, first, last):
    lengths = [0, 1, page * top, page * top + 1, 500, 1203]
    case = Case(kind, lengths, kv, dim, page, seed=13, slot_major=top == 5).upload()
    q = query_of(case, heads)
    want = case.expect_select(q, heads, top, first, last)
    got = case.select(q, heads, top, first, last)
    assert np.array_equal(got, want)
    check_attention(case, heads, q, selected=got, top=top)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (3, 3, 128), (34, 1, 40), (2, 2, 256)])
def test_selection_of_more_pages_than_there_are(gpu, kind, heads, kv, dim):
    """Runs of -1 before, between and behind the pages of a sequence, or only
    those; a page that no table has is reported from a run without others."""
    top = 260
    case = Case(kind, [300, 0, 17, 160, 299, 300], kv, dim, 16, seed=dim).upload()
    q = query_of(case, heads)
    chosen = case.select(q, heads, top, 1, 2)
    assert np.array_equal(chosen, case.expect_select(q, heads, top, 1, 2))
    check_attention(case, heads, q, selected=chosen, top=top)
    chosen[3] = np.roll(chosen[3], 200, axis=-1)
    for h in range(kv):
        chosen[4, h] = chosen[4, h][case.rng.permutation(top)]
    chosen[5] = -1
    check_attention(case, heads, q, selected=chosen, top=top)
    case.paged.check()
    chosen[5, kv - 1, 230] = 19  # one behind the last
    out, lse = case.attention(q, heads, selected=chosen, top=top)
    assert np.all(out[5] == 0) and np.all(np.isneginf(lse[5]))
    with pytest.raises(gpu.OutOfRange, match="page out of range"):
        case.paged.check()


@pytest.mark.parametrize("top", [4, 260])
def test_bad_length_beside_a_selection_of_nothing(gpu, top):
    case = Case("bf16", [100, 100], 2, 64, 16, seed=67)
    case.lengths[1] = 101
    case.upload()
    out, lse = case.attention(query_of(case, 4), 4, selected=np.full((2, 2, top), -1), top=top)
    assert np.all(out == 0) and np.all(np.isneginf(lse))
    with pytest.raises(gpu.OutOfRange, match="length out of range"):
        case.paged.check()


def test_select_ties_and_many_pages(gpu):
    """Pages of equal bounds go by their index; more pages than threads."""
    case = Case("bf16", [9000, 777], 2, 16, 1, seed=17)
    case.keys[:] = encode(np.round(decode(case.keys, "bf16")), "bf16")
    case.bounds[:, :, 0] = case.bounds[:, :, 1] = case.keys[:, :, 0]
    case.upload()
    q = np.round(query_of(case, 4))
    for top, first, last in ((64, 1, 2), (700, 0, 0), (1, 0, 0)):
        assert np.array_equal(case.select(q, 4, top, first, last),
                              case.expect_select(q, 4, top, first, last))
    case.bounds[:] = encode(np.float32(1.0), "bf16")
    case.upload()
    assert np.array_equal(case.select(q, 4, 64, 1, 2), case.expect_select(q, 4, 64, 1, 2))


@pytest.mark.parametrize("heads", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_select_equal_scores_of_unequal_pages(gpu, kind, heads):
    """Pages that agree in the bounds that a query meets, and differ in the
    others, score alike to the last bit: the lower ones are chosen."""
    case = Case(kind, [640], 1, 64, 16, seed=65)
    order = case.rng.permutation(40)
    best = case.rng.standard_normal(64)
    for c in order[:25]:
        case.bounds[case.table[0, c], 0, 1] = encode(best + 3, kind)
        case.bounds[case.table[0, c], 0, 0] = encode(-3 * case.rng.random(64), kind)
    case.upload()
    q = np.abs(query_of(case, heads)) * np.float32(1.1)
    want = case.expect_select(q, heads, 12, 0, 0)
    assert want[0, 0].tolist() == sorted(order[:25])[:12]
    assert np.array_equal(case.select(q, heads, 12, 0, 0), want)


def test_select_not_a_number_first(gpu):
    case = Case("f32", [320], 1, 16, 16, seed=19)
    case.bounds[case.table[0, 7], 0, 1, 3] = np.nan
    case.upload()
    got = case.select(query_of(case, 2), 2, 2, 0, 1)
    assert got.tolist() == [[[7, 19]]]


def select_by_definition(case, query, heads, top):
    """[batch][kv][top] from max(q lo, q hi) as written, no numbers first."""
    got = np.full((case.batch, case.kv, top), -1, np.int32)
    group, q = heads // case.kv, np.asarray(query, np.float64)
    for b, n in enumerate(case.lengths):
        count = -(-int(n) // case.page)
        for h in range(case.kv):
            bound = decode(case.bounds[case.table[b, :count], h], case.kind)
            mine = q[b, h * group:(h + 1) * group, None]
            with np.errstate(invalid="ignore"):
                score = np.maximum(mine * bound[:, 0], mine * bound[:, 1]).sum(-1)
            odd = np.isnan(score).any(0)
            best = np.where(np.isnan(score), -np.inf, score).max(0)
            rank = sorted(range(count), key=lambda c: (not odd[c], 0 if odd[c] else -best[c], c))
            chosen = sorted(rank[:top])
            got[b, h, :len(chosen)] = chosen
    return got


@pytest.mark.parametrize("heads,dim", [(1, 64), (2, 16), (3, 128), (4, 256), (5, 64), (8, 40),
                                       (16, 128), (20, 256)])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_select_infinite_bounds(gpu, kind, heads, dim):
    """An infinite bound counts where the query meets it and nowhere else: by
    the definition with queries of both signs, met from both sides (no number),
    by a component of 0 (no number), and beside a NaN."""
    case = Case(kind, [640, 170], 2, dim, 16, seed=77)
    inf = np.float32(np.inf)
    for b, n in enumerate(case.lengths):
        for c in range(-(-int(n) // 16)):
            for h in range(2):
                at = (case.table[b, c], h)
                d = case.rng.integers(dim, size=3)
                if c % 5 == 1:
                    case.bounds[(*at, 1, d[0])] = encode(inf, kind)
                if c % 5 == 2:
                    case.bounds[(*at, 0, d[0])] = encode(-inf, kind)
                if c % 10 == 3:
                    case.bounds[(*at, 0, d[:2])] = encode(-inf, kind)
                    case.bounds[(*at, 1, d[1:])] = encode(inf, kind)
                if c % 10 == 8:
                    case.bounds[(*at, slice(None), d[2])] = encode(-inf if h else inf, kind)
    case.bounds[case.table[1, 4], 1, 1, 5] = encode(np.float32(np.nan), kind)
    case.upload()
    for sign in (1, -1, 0):
        q = query_of(case, 2 * heads, seed=5 + sign)
        q = np.abs(q) * np.float32(sign) if sign else q
        if sign == 0:
            q[0, ::2, :3] = 0.0
        for top in (1, 3, 9, 20, 33):
            want = select_by_definition(case, q, 2 * heads, top)
            assert np.array_equal(case.select(q, 2 * heads, top, 0, 0), want), (sign, top)


@pytest.mark.parametrize("heads", [1, 4, 5, 8])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_select_bounds_that_the_query_does_not_meet(gpu, kind, heads):
    """Pages that agree in the bounds that a query meets score alike to the last
    bit, their others being infinite or not: the lower ones are chosen."""
    case = Case(kind, [640], 1, 64, 16, seed=79)
    order = case.rng.permutation(40)
    best = np.abs(case.rng.standard_normal(64))  # no upper bound below a lower one
    for i, c in enumerate(order[:25]):
        lo = -3 * case.rng.random(64)
        lo[case.rng.random(64) < 0.1 * (i % 3)] = -np.inf
        case.bounds[case.table[0, c], 0, 1] = encode(best + 3, kind)
        case.bounds[case.table[0, c], 0, 0] = encode(lo, kind)
    case.upload()
    q = np.abs(query_of(case, heads)) * np.float32(1.1)
    want = select_by_definition(case, q, heads, 12)
    assert want[0, 0].tolist() == sorted(order[:25])[:12]
    assert np.array_equal(case.select(q, heads, 12, 0, 0), want)


@pytest.mark.parametrize("heads", [2, 8])
def test_select_keys_beyond_the_type(gpu, heads):
    """Keys that the cache's type rounds to infinity, where the query has the
    other sign: the page's score is finite and not the best one."""
    case = Case("f16", [0], 1, 32, 8, seed=81, max_length=80).upload()
    k = case.rng.standard_normal((80, 1, 32)).astype(np.float32)
    k[20, 0, 4] = 70000.0  # page 2
    k[51] += 4.0           # page 6
    A = gpu.DeviceArray
    case.lengths = case.expect_append(k, k, [80])
    case.paged.append(case.seqs, A(like=k), A(like=k), None,
                      starts=A(like=np.array([0, 80], np.int32)), max_new=80)
    case.d["lengths"].upload(case.lengths)
    q = np.abs(query_of(case, heads)) + np.float32(0.1)
    q[..., 4] *= -1
    want = select_by_definition(case, q, heads, 3)
    assert 2 not in want[0, 0, :1] and 6 in want[0, 0]
    assert np.array_equal(case.select(q, heads, 3, 0, 0), want)
    assert np.array_equal(case.select(-q, heads, 1, 0, 0), [[[2]]])


def test_sparse_attention_of_a_callers_selection(gpu):
    """A page twice counts twice; -1 anywhere, and pages behind the sequence's
    end, count nothing; a page no table row has is reported."""
    case = Case("f32", [100, 100, 100], 1, 32, 16, seed=21).upload()
    q = query_of(case, 2)
    chosen = np.array([[[3, -1, 3, 0]], [[-1, -1, -1, -1]], [[6, 1, -1, -1]]], np.int32)
    check_attention(case, 2, q, selected=chosen, top=4)
    case.paged.check()
    chosen[1, 0, 2] = 1 << 30
    out, _ = case.attention(q, 2, selected=chosen, top=4)
    assert np.all(out[1] == 0)
    with pytest.raises(gpu.OutOfRange, match="page out of range"):
        case.paged.check()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,dim,page,budget,first,last,slot_major", [
    (2, 64, 16, 100, 4, 16, False), (3, 80, 24, 64, 0, 0, True), (1, 8, 1, 33, 1, 32, False),
    (2, 16, 300, 260, 0, 7, False), (2, 128, 128, 1, 0, 1, False), (1, 256, 7, 500, 0, 500, True),
])
def test_evict(gpu, kind, kv, dim, page, budget, first, last, slot_major):
    lengths = [0, 1, budget - 1, budget, budget + 1, budget + 40, 3 * budget + 5]
    case = Case(kind, lengths, kv, dim, page, seed=23, slot_major=slot_major)
    # heavy tails, rows without weight, positions as earlier evictions leave them
    case.weights[:] = np.exp(3 * case.rng.standard_normal(case.weights.shape))
    case.weights[case.rng.random(case.weights.shape) < 0.2] = 0.0
    for b in range(case.batch):
        for h in range(kv):
            case.positions[b, h] = 3 * case.rng.permutation(case.max_length)
    check_evict(case, budget, first, last)


def check_evict(case, budget, first=0, last=0):
    case.upload()
    new = case.expect_evict(budget, first, last)
    case.evict(budget, first, last)
    assert np.array_equal(case.new_lengths(), new)
    for name in ("weights", "positions", "bounds"):
        assert same(case.fetch(name), getattr(case, name)), name
    for name in ("keys", "values"):
        assert same(case.pool(name), getattr(case, name)), name
    case.paged.check()


def test_evict_ties_and_not_numbers(gpu):
    case = Case("f16", [900, 450], 2, 16, 16, seed=25)
    case.weights[0] = 0.5                     # all equal: the first rows stay
    case.weights[1] = np.round(case.weights[1] * 4) / 4
    case.weights[1, 0, ::3] = np.nan          # below all others
    case.weights[1, 1, ::5] = np.inf
    case.weights[1, 1, 1::5] = -np.inf
    case.weights[1, 1, 2::5] = -0.0
    check_evict(case, 300, 2, 10)


@pytest.mark.parametrize("more", [1, 3, 257])
def test_evict_a_few_of_many(gpu, more):
    """Budgets just below the longest sequence, and above every one."""
    lengths = [700 + more, 700, 699 + more, 12]
    case = Case("bf16", lengths, 2, 16, 16, seed=more, max_length=700 + more)
    case.weights[:] = np.exp(case.rng.standard_normal(case.weights.shape))
    check_evict(case, 700, 1, 5)
    check_evict(case, 1 << 30, 1, 5)


def test_evict_long(gpu):
    """Many more rows than threads, and twice in a row."""
    case = Case("bf16", [20000, 15001], 1, 8, 64, seed=27)
    case.weights[:] = np.exp(case.rng.standard_normal(case.weights.shape))
    check_evict(case, 4096, 4, 512)
    case.lengths = case.new_lengths()
    check_evict(case, 4000, 4, 512)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,dim,page,slot_major", [
    (2, 64, 16, False), (4, 128, 32, True), (1, 8, 1, False), (3, 80, 24, False),
    (2, 256, 300, True)])
def test_append_ragged(gpu, kind, kv, dim, page, slot_major):
    lengths = [0, 1, 15, 16, 17, 250, 3, 0]
    counts = [1, 40, 1, 16, 0, 333, 2, 0]
    case = Case(kind, lengths, kv, dim, page, seed=29, slot_major=slot_major, room=340).upload()
    rows = sum(counts) + 5  # source rows behind the last sequence's
    k = case.rng.standard_normal((rows, kv, dim)).astype(np.float32)
    v = case.rng.standard_normal((rows, kv, dim)).astype(np.float32)
    firsts = np.arange(1000, 1000 + 50 * len(counts), 50, dtype=np.int32)
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    new = case.expect_append(k, v, counts, firsts=firsts)
    A = gpu.DeviceArray
    case.paged.append(case.seqs, A(like=k), A(like=v), case.d["new_lengths"], starts=A(like=starts),
                      max_new=333, history=case.history, first_positions=A(like=firsts))
    gpu.synchronize()
    check_append(case, new)


def check_append(case, new):
    assert np.array_equal(case.new_lengths(), new)
    for name in ("weights", "positions", "bounds"):
        assert same(case.fetch(name), getattr(case, name)), name
    for name in ("keys", "values"):
        assert same(case.pool(name), getattr(case, name)), name
    case.paged.check()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,dim", [(2, 16), (4, 64), (1, 40), (32, 128), (2, 256)])
def test_append_tokens(gpu, kind, kv, dim):
    """One row each, out of fused rows [q | k | v], with rounding ties, values
    beyond fp16, signed zeros, subnormals and infinities among the values."""
    case = Case(kind, [0, 5, 15, 16, 63], kv, dim, 16, seed=31, room=1).upload()
    fused = case.rng.standard_normal((case.batch, 3, kv, dim)).astype(np.float32)
    odd = np.array([1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, -0.0,
                    70000.0, 65519.9, 2.0 ** -25, 3 * 2.0 ** -25, 1e-40, np.inf, -np.inf,
                    3.4e38, -1.0], np.float32)
    flat = fused[:, 2].reshape(case.batch, -1).copy()
    flat[1, :14], flat[2, -14:] = odd, odd
    fused[:, 2] = flat.reshape(case.batch, kv, dim)
    whole = gpu.DeviceArray(like=fused)

    class Part:
        def __init__(self, i):
            self.ptr = whole.ptr.value + 4 * i * kv * dim
            self.nbytes = whole.nbytes - 4 * i * kv * dim

    new = case.expect_append(fused[:, 1], fused[:, 2], [1] * 5)
    case.paged.append(case.seqs, Part(1), Part(2), case.d["new_lengths"], history=case.history,
                      row_stride=3 * kv * dim, head_stride=dim)
    gpu.synchronize()
    check_append(case, new)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("kv,dim,row_stride,head_stride", [
    (3, 32, 3 * 3 * 32, 0), (3, 32, 0, 32), (4, 64, 4 * 64 + 8, 0), (3, 32, 32, 160),
    (1, 64, 0, 8), (2, 16, 0, 0)])
def test_append_strides(gpu, kv, dim, row_stride, head_stride, ragged):
    """One stride without the other, heads before rows, and heads of one."""
    counts = [1, 2, 2] if ragged else [1, 1, 1]
    case = Case("f32", [0, 7, 16], kv, dim, 16, seed=75, room=2).upload()
    rows = sum(counts)
    row, head = row_stride or kv * dim, head_stride or dim
    flat = case.rng.standard_normal(2 * (rows * row + kv * head)).astype(np.float32)
    at = (np.arange(rows)[:, None, None] * row + np.arange(kv)[:, None] * head + np.arange(dim))
    k, v = flat[at], flat[at + 4]
    new = case.expect_append(k, v, counts)
    A = gpu.DeviceArray
    whole = A(like=flat)

    class Part:
        def __init__(self, first):
            self.ptr = whole.ptr.value + 4 * first
            self.nbytes = 4 * (flat.size - first)

    starts = A(like=np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
    case.paged.append(case.seqs, Part(0), Part(4), case.d["new_lengths"],
                      starts=starts if ragged else None, max_new=max(counts),
                      history=case.history, row_stride=row_stride, head_stride=head_stride)
    gpu.synchronize()
    check_append(case, new)


def test_append_not_a_number_shows_in_the_bounds(gpu):
    case = Case("f32", [3, 0], 1, 16, 8, seed=33, room=2).upload()
    k = np.ones((2, 1, 16), np.float32)
    k[0, 0, 4] = k[1, 0, 5] = np.nan
    A = gpu.DeviceArray
    case.paged.append(case.seqs, A(like=k), A(like=k), case.d["new_lengths"])
    gpu.synchronize()
    for b, d in ((0, 4), (1, 5)):
        nan = np.isnan(case.fetch("bounds")[case.table[b, 0], 0])
        assert np.all(nan[:, d]) and nan.sum() == 2


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(3, 1, 32), (8, 1, 64), (2, 2, 96), (17, 1, 128),
                                          (5, 1, 256)])
def test_attention_room_for_long_sequences(gpu, kind, heads, kv, dim):
    """Calls that allow for millions of rows (and read past the caches) over
    short sequences: the table's entries behind them are not followed."""
    case = Case(kind, [700, 0, 33, 1025], kv, dim, 32, seed=59).upload()
    q = query_of(case, heads)
    out, lse, _, tol, _ = case.expect_attention(q, heads)
    most = (256 << 20) // (kv * dim * 2 * (4 if kind == "f32" else 2)) // 4
    width = -(-most // 32)
    table = np.full((4, width), -1, np.int32)
    table[:, :case.width] = case.table
    A = gpu.DeviceArray
    d_table = A(like=table)
    seqs = gpu.PagedBatch(d_table, width, case.d["lengths"], 4, most)
    need = case.paged.attention_workspace(seqs, heads)
    work = A(like=np.full(need, 0xff, np.uint8))
    dq, do, dl = A(like=q), A(out.size * 4), A(lse.size * 4)
    case.paged.attention(seqs, dq, do, heads, lse=dl, workspace=work)
    gpu.synchronize()
    got = do.download(np.float32, out.size).reshape(out.shape)
    assert np.all(np.abs(got - out) <= tol)
    case.paged.check()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_attention_queries_that_are_not_finite(gpu, kind):
    """A query with a NaN, or with an infinity (whose products with keys of both
    signs are both infinities), gives no number for its own head alone; one
    whose scores are all minus infinity gives zeros."""
    case = Case(kind, [40], 2, 32, 16, seed=61)
    for h in range(2):
        for i in range(40):
            row = decode(case.keys[case.table[0, i // 16], h, i % 16], kind)
            row[7] = abs(row[7]) + 0.5
            case.keys[case.table[0, i // 16], h, i % 16] = encode(row, kind)
    case.upload()
    q = query_of(case, 8)
    q[0, 1, 3], q[0, 2, 7], q[0, 5, 7], q[0, 6, 2] = np.nan, np.inf, -np.inf, np.inf
    got, lse = case.attention(q, 8)
    plain = [0, 3, 4, 7]
    out, want, _, tol, _ = case.expect_attention(np.nan_to_num(q, posinf=0, neginf=0), 8)
    assert np.all(np.abs(got - out)[0, plain] <= tol[0, plain])
    assert np.all(np.isnan(got[0, [1, 2, 6]]))
    assert np.all(got[0, 5] == 0) and np.isneginf(lse[0, 5])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [1.0, 1e5, 1e9, 1e30])
def test_attention_infinite_queries_of_any_size(gpu, kind, size):
    """An infinite component decides whatever the size of the finite ones."""
    case = Case(kind, [40, 300], 2, 64, 16, seed=85)
    rows = decode(case.keys, kind)
    rows[..., 7] = np.abs(rows[..., 7]) + 0.5
    case.keys[:] = encode(rows, kind)
    case.upload()
    q = query_of(case, 4) * np.float32(size)
    q[0, 0, 7], q[1, 1, 7], q[0, 3, 7] = -np.inf, -np.inf, np.inf
    got, lse = case.attention(q, 4)
    for b, h in ((0, 0), (1, 1)):
        assert np.all(got[b, h] == 0) and np.isneginf(lse[b, h])
    assert np.all(np.isnan(got[0, 3]))
    rest = [(0, 1), (0, 2), (1, 0), (1, 2), (1, 3)]
    out, _, _, tol, _ = case.expect_attention(np.nan_to_num(q, posinf=0, neginf=0), 4)
    for b, h in rest:
        assert np.all(np.abs(got - out)[b, h] <= tol[b, h])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_attention_values_that_are_not_finite(gpu, kind):
    """An infinite or NaN value shows in its component of the KV head's results
    and nowhere else."""
    case = Case(kind, [40], 2, 32, 16, seed=63)
    out, _, _, tol, _ = case.expect_attention(query_of(case, 4), 4)
    case.values[case.table[0, 1], 1, 2, 9] = encode(np.array(np.inf), kind)
    case.values[case.table[0, 2], 1, 5, 20] = encode(np.array(np.nan), kind)
    case.upload()
    got, _ = case.attention(query_of(case, 4), 4)
    odd = np.zeros_like(got, bool)
    odd[0, 2:, [9, 20]] = True
    assert np.array_equal(~np.isfinite(got), odd)
    assert np.all(np.abs(got - out)[~odd] <= tol[~odd])
