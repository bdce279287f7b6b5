"""What calls over page pools and beams write may share no memory with what they read, or
with one another: each refusal, and the addresses next to it, on a host without a GPU."""
import pytest

import nutllm_amd as nut
from test_cpu_serving import (At, beams, compact, gather, pool, pytestmark, reaches, refused,  # noqa: F401
                              reorder, select, table)

BASE = 1 << 16  # a table of 3 x 8 entries, its lengths 4,096 bytes on, held pages 8,192


@pytest.mark.parametrize("copies", [BASE - 56, BASE, BASE + 92, BASE + 8192, BASE + 8200,
                                    4096 - 56, 4096, 4096 + 36])
def test_compact_copies_over_table_or_counts(copies):
    refused("copies, counts and table overlap", compact, copies=At(copies))


@pytest.mark.parametrize("copies", [BASE - 60, BASE + 96, BASE + 8192 + 12, 4096 - 60, 4096 + 40])
def test_compact_copies_beside_them(copies):
    reaches(compact, copies=At(copies))


def test_compact_counts_over_table():
    for refs in (BASE - 36, BASE + 92, BASE + 8192 - 36, BASE + 8200):
        refused("copies, counts and table overlap", compact, pool(At(refs)))
    for refs in (BASE - 40, BASE + 96, BASE + 8192 + 12):
        reaches(compact, pool(At(refs)))
    refused("copies, counts and table overlap", compact, None, table(held=At(BASE + 88)))


def test_reorder_counts_over_a_table():
    new = 1 << 18
    for refs in (BASE - 36, BASE + 92, BASE + 4096, BASE + 8200, new, new + 4096, new + 8192,
                 1 << 24, (1 << 24) + 4096 + 32):
        refused("counts overlap a table", reorder, pool(At(refs)))
    for refs in (BASE - 40, BASE + 96, new - 40, new + 96, (1 << 24) + 12, (1 << 24) + 4096 + 36):
        reaches(reorder, pool(At(refs)))


NEW = {"scores": 0, "lengths": 4096, "ended": 8192}


@pytest.mark.parametrize("one", [*NEW, "parents", "tokens"])
@pytest.mark.parametrize("two", [*NEW, "parents", "tokens"])
@pytest.mark.parametrize("by,over", [(-32, False), (-28, True), (0, True), (28, True),
                                     (32, False)])
def test_select_outputs_over_one_another(one, two, by, over):
    if one == two:
        return
    at = {**{k: (1 << 22) + v for k, v in NEW.items()}, "parents": 1 << 24, "tokens": 1 << 25}
    at[two] = at[one] + by
    new = beams(1 << 22, **{k: At(at[k]) for k in NEW})
    args = (None, new), dict(parents=At(at["parents"]), tokens=At(at["tokens"]))
    if over:
        refused("overlaps itself", select, *args[0], **args[1])
    else:
        reaches(select, *args[0], **args[1])


@pytest.mark.parametrize("dtype,size", [(nut.F32, 4), (nut.F16, 2)])
@pytest.mark.parametrize("stride", [1000, 1100])
def test_select_outputs_over_the_logits(dtype, size, stride):
    """Eight rows of 1,000 logits."""
    logits, end = 1 << 26, (1 << 26) + (7 * stride + 1000) * size
    kw = dict(logits=At(logits), dtype=dtype, row_stride=stride)
    for at in (logits - 28, logits, end - 4):
        refused("overlaps the logits", select, tokens=At(at), **kw)
        refused("overlaps the logits", select, None, beams(1 << 22, scores=At(at)), **kw)
    for at in (logits - 32, end):
        reaches(select, tokens=At(at), **kw)


def test_gather_over_the_parents():
    to = 1 << 24  # three rows of 64 bytes
    for at in (to - 8, to, to + 188):
        refused("overlap the parents", gather, parents=At(at))
    for at in (to - 12, to + 192):
        reaches(gather, parents=At(at))
