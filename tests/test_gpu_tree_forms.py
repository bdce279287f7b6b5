"""The forms of tree attention (few query rows, two tiles of them, many with rows in
shared memory, rows read past the caches) at the masks, values, strides and bad
arguments where each can go wrong. Which form a call takes is its sizes' matter: the
workspace that it asks for shows that a test reaches the form that it is for."""
import numpy as np
import pytest

from paged_case import decode, encode
from serving_case import TreeCase, attend64, dev

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f16", "bf16"]
FORMS = ["tree", "staged"]
MANY = 40000  # rows that a table may hold, far more than any sequence does
# not numbers, by their bits: the payload in low bits alone, quiet ones, both signs
NANS = {"f32": [0x7f800001, 0xff80ffff, 0x7fc00000], "f16": [0x7c01, 0xfe00],
        "bf16": [0x7f81, 0xffc0]}
BITS = {"f32": np.uint32, "f16": np.uint16, "bf16": np.uint16}


def wide(c, max_length=MANY):
    """The case behind a table that could hold `max_length` rows a sequence."""
    case = c.case
    width = -(-max_length // case.page)
    more = np.full((case.batch, width - case.width), -1, np.int32)
    case.table, case.width = np.concatenate([case.table, more], 1), width
    case.max_length = max_length
    return c


def _up(n):
    return -(-n // 256) * 256


def staged_bytes(kind, dim, batch):
    """Two parts of 64 query rows for every share, and the stages before each sequence."""
    groups = 3 if dim <= 64 else (3 if dim <= 128 else 2) - (kind == "f32")
    shares = 256 * groups
    return _up(shares * 128 * dim * 4) + _up(shares * 128 * 8) + _up((batch + 1) * 8)


def tree_runs(columns, most):
    """Runs of a sequence: as long as make 1,024 workgroups, or down to 128 rows."""
    run = -(-most // 128) * 128
    while run > 128 and columns * -(-most // run) < 1024:
        run = -(-(run // 2) // 128) * 128
    return -(-most // run)


def tree_bytes(c, tiles):
    """The runs' parts, where a workgroup takes `tiles` tiles of 16 query rows."""
    queries = c.most * (c.heads // c.kv)
    runs = tree_runs(len(c.held) * c.kv * -(-queries // (16 * tiles)), c.case.max_length)
    parts = c.total * c.heads * runs
    return 0 if runs == 1 else _up(parts * c.dim * 4) + _up(parts * 8)


def work_of(c):
    return c.case.paged.tree_attention_workspace(c.seqs, c.draft, c.heads)


def rows_at(c, b, h, rows):
    """Keys and values of some rows of a sequence."""
    page, slot = c.case.table[b, rows // c.case.page], rows % c.case.page
    return [decode(p[page, h, slot], c.kind) for p in (c.case.keys, c.case.values)]


def ready(c, form):
    """The case uploaded, with a table as wide as its form asks for."""
    if form == "staged":
        wide(c)
    c.upload()
    staged = work_of(c) == staged_bytes(c.kind, c.dim, len(c.held))
    assert staged == (form == "staged")
    return c


# ------------------------------------------------- two tiles of query rows --

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [8, 32, 40, 64, 80, 96, 120, 128, 136, 256])
@pytest.mark.parametrize("heads,kv,most,order", [(8, 1, 4, False), (16, 2, 3, True),
                                                 (1, 1, 27, True), (6, 2, 10, False),
                                                 (2, 2, 32, False)])
def test_two_tiles(gpu, kind, dim, heads, kv, most, order):
    """17 to 32 query rows a KV head, many parts joined; sequences of every few nodes,
    so that one tile has all of a workgroup's rows, and the other one row or none."""
    held = [300, 0, 1, 33, 64, 127, 129, 40]
    counts = [most, most, 1, 2, most - 1, 0, most // 2 + 1, most]
    c = wide(TreeCase(kind, held, counts, kv, dim, 16, heads, seed=dim, slot_major=order, lead=1,
                      trail=2))
    c.upload()
    assert work_of(c) == tree_bytes(c, 2) != tree_bytes(c, 1)
    c.check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads", [(64, 8), (24, 8), (128, 6), (256, 7)])
def test_two_tiles_of_short_rows(gpu, kind, dim, heads):
    """So many sequences that nothing is split: the results come from the one launch."""
    rng = np.random.default_rng(dim)
    held = rng.integers(0, 60, 530).tolist()
    counts = rng.integers(0, 5, 530).tolist()
    counts[0], held[1] = 4, 124
    c = TreeCase(kind, held, counts, 1, dim, 32, heads, seed=7, max_length=128).upload()
    assert work_of(c) == 0 and 530 * 2 > 1024  # of 16 query rows and 128 rows: two tiles
    c.check()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_two_tiles_over_pieces(gpu, kind):
    """More rows in a run than offsets are kept of at once."""
    held, counts = [3] * 1030, [1] * 1030
    held[1], held[700], counts[1], counts[700] = 2000, 1500, 4, 3
    c = TreeCase(kind, held, counts, 1, 16, 2048, 8, seed=1, max_length=2048).upload()
    assert work_of(c) == 0  # one run of 2,048 rows
    c.check()


@pytest.mark.parametrize("kind", KINDS)
def test_two_tiles_any_mask(gpu, kind):
    rng = np.random.default_rng(4)
    counts, held = [27, 20, 32, 5], [0, 9, 31, 0]
    sees = [rng.random((m, m)) < 0.3 for m in counts]
    sees[0][5], sees[1][:], sees[3][:] = False, False, False
    c = wide(TreeCase(kind, held, counts, 2, 64, 16, 2, seed=2, sees=sees), 2 * MANY)
    c.upload()
    assert work_of(c) == tree_bytes(c, 2) != tree_bytes(c, 1)
    c.check()


# --------------------------------------------------- rows in shared memory --

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads", [(64, 8), (80, 4), (128, 2), (256, 2), (24, 3)])
def test_staged_any_mask(gpu, kind, dim, heads):
    """Masks that are no tree's: random ones, none, and nothing where no row is held."""
    rng = np.random.default_rng(dim)
    counts, held = [90, 7, 33, 5, 70], [0, 9, 31, 0, 200]
    sees = [rng.random((m, m)) < 0.3 for m in counts]
    sees[0][5], sees[1][:], sees[3][:], sees[4][:] = False, False, False, False
    ready(TreeCase(kind, held, counts, 1, dim, 16, heads, seed=2, sees=sees), "staged").check()


@pytest.mark.parametrize("kind", KINDS)
def test_staged_strided_queries(gpu, kind):
    """Query rows with others' components between them; no log-sums asked for."""
    c = ready(TreeCase(kind, [50, 3, 140], [49, 14, 60], 2, 64, 16, 4, seed=3), "staged")
    flat = np.full((c.total, 4 * 64 + 20), np.nan, np.float32)
    flat[:, :256] = c.query.reshape(c.total, 256)
    c.check(query=dev(flat, np.float32), query_stride=276)
    c.out.upload(np.full(c.out.nbytes // 4, 7.0, np.float32))
    c.case.paged.tree_attention(c.seqs, c.draft, c.d_query, c.out, 4, workspace=c.work)
    out, _, tol, _ = c.expect()
    assert np.all(np.abs(c.results()[0] - out) <= tol)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", ["starts", "total", "most", "length", "longest", "page"])
def test_staged_of_what_it_cannot_follow(gpu, kind, bad):
    """The other sequences' results stand, and the check says what was wrong."""
    c = ready(TreeCase(kind, [40, 20, 90], [46, 35, 57], 2, 64, 16, 4, seed=6, trail=60), "staged")
    out, lse, tol, tol_lse = c.expect()
    mine, last = slice(c.starts[1], c.starts[2]), slice(c.starts[2], c.starts[3])
    message, starts = "rows out of range", c.starts.copy()
    if bad == "starts":  # sequence 1 begins behind its end, 0 ends there: too many nodes
        starts[1] = starts[2] + 3
        c.d_starts.upload(starts)
        out[:last.start], lse[:last.start] = 7.0, 7.0
    elif bad == "total":
        starts[3] = c.total + 1
        c.d_starts.upload(starts)
        out[last], lse[last] = 7.0, 7.0
    elif bad == "most":
        c.draft.view.most = 50
        out[last], lse[last] = 7.0, 7.0
    elif bad in ("length", "longest"):
        held = np.array(c.held, np.int32)
        held[1] = -1 if bad == "length" else c.case.max_length - 34
        c.d_held.upload(held)
        out[mine], lse[mine], message = 0.0, -np.inf, "length out of range"
    else:  # rows 16 to 31 of sequence 1 are on a page that is not there
        c.case.table[1, 1] = c.case.pages
        c.case.d["table"].upload(c.case.table)
        message = "page out of range"
        rows = np.concatenate([np.arange(16), np.arange(32, 55)])
        for h in range(4):
            k, v = rows_at(c, 1, h // 2, rows)
            for i in range(35):
                at = (rows < 20) | ((rows >= 32) & c.sees[1][i][np.maximum(rows - 20, 0)])
                row = c.starts[1] + i
                out[row, h], lse[row, h], tol[row, h], tol_lse[row, h] = attend64(
                    c.query[row, h], k[at], v[at], 1 / 8)
    got, got_lse = c.attention()
    assert np.all(np.abs(got - out) <= tol)
    empty = np.isneginf(lse)
    assert np.array_equal(np.isneginf(got_lse), empty)
    assert np.all(np.abs(got_lse[~empty] - lse[~empty]) <= tol_lse[~empty])
    with pytest.raises(gpu.OutOfRange, match=message):
        gpu.check_status(c.status)
    gpu.check_status(c.status)


# ------------------------------------------------ what is no finite number --

def put(c, pool, b, row, component, value=None, bits=None):
    """One component of a row of the sequence, in every KV head."""
    a = getattr(c.case, pool)
    at = (c.case.table[b, row // c.case.page], slice(None), row % c.case.page, component)
    if bits is None:
        a[at] = encode(np.array([value]), c.kind)[0]
    else:
        a.view(BITS[c.kind])[at] = bits


def seen_rows(c, b, i):
    return np.concatenate([np.arange(c.held[b]),
                           c.held[b] + np.nonzero(c.sees[b][i])[0]]).astype(int)


def bare(kind, form, dim, heads):
    """Two sequences, many of whose rows are far from the drafted ones."""
    return TreeCase(kind, [200, 70], [45, 36], 1, dim, 16, heads, seed=dim)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim,heads", [(64, 4), (80, 2), (128, 1), (256, 2), (8, 3)])
@pytest.mark.parametrize("row", [5, 203])
@pytest.mark.parametrize("sign", [1, -1])
def test_infinite_keys(gpu, kind, form, dim, heads, row, sign):
    """A key with one infinite component, of a row that the sequence held or of node 3:
    where it makes the score minus infinity the row has no part, where it makes it
    infinite the result is no number, and nodes that do not see it are as ever."""
    c = bare(kind, form, dim, heads)
    put(c, "keys", 0, row, 5, sign * np.inf)
    ready(c, form)
    got, lse = c.attention()
    for b in range(2):
        k, v = rows_at(c, b, 0, np.arange(c.held[b] + c.counts[b]))
        for i in range(c.counts[b]):
            at, mine = seen_rows(c, b, i), c.starts[b] + i
            for h in range(heads):
                if b == 0 and row in at and c.query[mine, h, 5] * sign > 0:
                    assert np.all(np.isnan(got[mine, h])) and not np.isfinite(lse[mine, h])
                    continue
                rest = at[at != row] if b == 0 else at
                want, want_lse, tol, tol_lse = attend64(c.query[mine, h], k[rest], v[rest],
                                                        dim ** -0.5)
                assert np.all(np.abs(got[mine, h] - want) <= tol)
                assert abs(lse[mine, h] - want_lse) <= tol_lse


@pytest.mark.parametrize("kind,bits", [(k, b) for k in KINDS for b in NANS[k]])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim,heads", [(64, 4), (80, 2), (128, 1), (256, 2)])
@pytest.mark.parametrize("row", [5, 203])
def test_keys_that_are_no_numbers(gpu, kind, bits, form, dim, heads, row):
    """Whatever its bits, a key that is no number makes the results no numbers of the
    nodes that see it, and of no others."""
    c = bare(kind, form, dim, heads)
    out, want_lse, tol, tol_lse = c.expect()
    put(c, "keys", 0, row, 5, bits=bits)
    got, lse = ready(c, form).attention()
    for b in range(2):
        for i in range(c.counts[b]):
            mine = c.starts[b] + i
            if b == 0 and row in seen_rows(c, b, i):
                assert np.all(np.isnan(got[mine])) and np.all(np.isnan(lse[mine]))
            else:
                assert np.all(np.abs(got[mine] - out[mine]) <= tol[mine])
                assert np.all(np.abs(lse[mine] - want_lse[mine]) <= tol_lse[mine])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim,heads", [(64, 4), (80, 2), (128, 1), (256, 2), (8, 3)])
def test_queries_that_are_not_finite(gpu, kind, form, dim, heads):
    """A query that is no number, one that makes every score minus infinity, one that makes
    them infinite: their nodes' results alone are none, nothing, and none."""
    c = bare(kind, form, dim, heads)
    keys = c.case.keys  # component 2 is below 0 in every key
    keys[..., 2] = encode(-np.abs(decode(keys[..., 2], kind)) - 0.25, kind)
    none, nothing, all_of_it = c.starts[0] + 7, c.starts[0] + 20, c.starts[1] + 3
    out, want_lse, tol, tol_lse = c.expect()
    c.query.view(np.uint32)[none, heads - 1, 5] = 0x7f800001
    c.query[nothing, :, 2], c.query[all_of_it, :, 2] = np.inf, -np.inf
    got, lse = ready(c, form).attention()
    assert np.all(np.isnan(got[none, heads - 1])) and np.isnan(lse[none, heads - 1])
    assert np.all(got[nothing] == 0) and np.all(np.isneginf(lse[nothing]))
    assert np.all(np.isnan(got[all_of_it])) and not np.any(np.isfinite(lse[all_of_it]))
    rest = np.ones((c.total, heads), bool)
    rest[none, heads - 1] = rest[nothing] = rest[all_of_it] = False
    assert np.all((np.abs(got - out) <= tol)[rest])
    assert np.all((np.abs(lse - want_lse) <= tol_lse)[rest])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim,heads", [(64, 4), (80, 2), (128, 1), (256, 2), (8, 3)])
@pytest.mark.parametrize("row", [5, 203])
@pytest.mark.parametrize("what", ["inf", "-inf", "nan"])
def test_values_that_are_not_finite(gpu, kind, form, dim, heads, row, what):
    """One component of a value, of a row that the sequence held or of node 3: that
    component of what sees it is not finite, the others and the log-sums are as ever."""
    c = bare(kind, form, dim, heads)
    out, want_lse, tol, tol_lse = c.expect()
    at = 6
    if what == "nan":
        put(c, "values", 0, row, at, bits=NANS[kind][0])
    else:
        put(c, "values", 0, row, at, float(what))
    got, lse = ready(c, form).attention()
    assert np.all(np.abs(lse - want_lse) <= tol_lse)
    rest = np.arange(dim) != at
    assert np.all(np.abs(got - out)[..., rest] <= tol[..., rest])
    for b in range(2):
        for i in range(c.counts[b]):
            mine = c.starts[b] + i
            if b != 0 or row not in seen_rows(c, b, i):
                assert np.all(np.abs(got[mine, :, at] - out[mine, :, at]) <= tol[mine, :, at])
            elif what == "nan":
                assert np.all(np.isnan(got[mine, :, at]))
            else:  # weights of 0 in a limb may make it no number
                assert not np.any(np.isfinite(got[mine, :, at]))
                if row > c.held[0]:  # drafted: added one by one
                    assert np.all(got[mine, :, at] == float(what))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads", [(64, 4), (80, 2), (128, 1), (256, 2)])
def test_staged_rows_that_are_not_finite(gpu, kind, dim, heads):
    """Whole drafted rows, infinite or no numbers: nodes that do not see them have their
    results as ever; those that see them do not have finite ones."""
    c = TreeCase(kind, [21, 0], [60, 39], 1, dim, 16, heads, seed=dim)
    bad = {0: [(3, "values", np.nan), (17, "values", np.inf), (18, "keys", np.nan),
               (30, "values", -np.inf), (39, "keys", np.inf)], 1: [(4, "values", np.nan)]}
    out, want_lse, tol, tol_lse = c.expect()
    for b, rows in bad.items():
        for i, name, x in rows:
            put(c, name, b, c.held[b] + i, slice(None), x)
    got, lse = ready(c, "staged").attention()
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


# ------------------------------------------------------ large and small ones --

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim,heads", [(32, 4), (80, 2), (128, 3)])
def test_large_scores(gpu, kind, form, dim, heads):
    c = TreeCase(kind, [5, 77, 260], [36, 40, 18], 1, dim, 16, heads, seed=8, sigma=30.0)
    c.query *= 13.0
    ready(c, form).check()
    c.check(scale=0.0)
    c.check(scale=-0.25)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [64, 80, 128])
def test_components_of_all_sizes(gpu, kind, form, dim):
    """Components as far apart as the types hold, those of keys and queries against one
    another, so that every one has a part in the scores; in the values each its own."""
    c = TreeCase(kind, [40, 150], [40, 33], 1, dim, 16, 2, seed=dim)
    most = 4 if kind == "f16" else 60
    by = np.exp2(np.random.default_rng(dim).integers(-most, most + 1, dim))
    for name in ("keys", "values"):
        setattr(c.case, name, encode(decode(getattr(c.case, name), kind) * by, kind))
    c.query = (c.query / by).astype(np.float32)
    ready(c, form).check()


# ---------------------------------------------------------- past the caches --

@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dim,heads,kv", [(64, 2, 2), (80, 1, 1), (128, 4, 2), (256, 1, 1),
                                          (24, 1, 1), (96, 2, 2)])
def test_rows_past_the_caches(gpu, kind, dim, heads, kv):
    """One block of query rows a KV head over what may be 128 MiB of rows: read past the
    caches' replacement, with results that are those of a call of less, to the last bit."""
    most = 64 * kv // heads
    held, counts = [700, 0, 64, 33], [most, most // 2, 1, most - 1]
    rows = (128 << 20) // (len(held) * kv * dim * 2 * 2)
    got = []
    for max_length in (rows, rows - 1):
        c = wide(TreeCase(kind, held, counts, kv, dim, 16, heads, seed=dim, trail=1), max_length)
        c.upload()
        assert work_of(c) == staged_bytes(kind, dim, len(held))
        got.append(c.attention())
        c.check(got[-1])
    for a, b in zip(*got):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
