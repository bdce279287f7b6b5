"""The forms of tree attention (few query rows, two tiles of them, many with rows in
shared memory, rows read past the caches) at the masks, values, strides and bad
arguments where each can go wrong. Which form a call takes is its sizes' matter: the
workspace that it asks for shows that a test reaches the form that it is for."""
import numpy as np
import pytest

from paged_case import decode, encode
from serving_case import TreeCase, attend64

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
