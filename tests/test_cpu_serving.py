"""What the entry points of draft trees, page pools and beam search refuse before
anything is launched, on a host without a GPU: each refusal's message, and that
the arguments next to it come through to the device (and fail there, loudly,
where there is none)."""
import ctypes as C
import os
import subprocess

import pytest

import nutllm_amd as nut


class At:
    """A buffer that no call here may touch."""

    def __init__(self, address=4096, nbytes=1 << 30):
        self.ptr, self.nbytes = address, nbytes


def _no_gpu():
    try:
        return nut.device_count() == 0
    except nut.DeviceError:
        return True


pytestmark = pytest.mark.skipif(not _no_gpu(), reason="a GPU is visible")
NONE = At(None)


def paged(**kw):
    a = {**dict(keys=At(), values=At(), pages=10, page_size=16, kv_heads=2, head_dim=64,
                dtype=nut.BF16, bounds=At()), **kw}
    return nut.PagedKV(a.pop("keys"), a.pop("values"), a.pop("pages"), a.pop("page_size"),
                       a.pop("kv_heads"), a.pop("head_dim"), a.pop("dtype"),
                       bounds=a.pop("bounds"), **a)


def seqs(**kw):
    a = {**dict(pages=At(), stride=4, lengths=At(8192), batch=3, most=64), **kw}
    return nut.PagedBatch(a["pages"], a["stride"], a["lengths"], a["batch"], a["most"])


def tree(**kw):
    a = {**dict(parents=At(), mask=At(), most=40, total=100, batch=3, starts=At()), **kw}
    return nut.DraftTree(a.pop("parents"), a.pop("mask"), a.pop("most"), a.pop("total"),
                         a.pop("batch"), **a)


def table(base=1 << 16, **kw):
    a = {**dict(pages=At(base), stride=8, lengths=At(base + 4096), held=At(base + 8192), batch=3),
         **kw}
    return nut.PageTable(a["pages"], a["stride"], a["lengths"], a["held"], a["batch"])


def pool(refs=At(), pages=10, page_size=16):
    return nut.PagePool(refs, pages, page_size)


def beams(base=1 << 20, **kw):
    a = {**dict(scores=At(base), requests=2, beams=4, lengths=At(base + 4096),
                ended=At(base + 8192)), **kw}
    return nut.BeamState(a["scores"], a["requests"], a["beams"], lengths=a["lengths"],
                         ended=a["ended"])


def build(d=None, **kw):
    (d or tree()).build(depths=At(), **kw)


def accept(d=None, s=None, **kw):
    a = dict(tokens=At(), chosen=At(), path=At(), counts=At(), new_lengths=At())
    a.update(kw)
    (d or tree()).accept(s or seqs(), a.pop("tokens"), a.pop("chosen"), a.pop("path"),
                         a.pop("counts"), **a)


def attention(d=None, s=None, kv=None, **kw):
    a = dict(query=At(), out=At(), heads=8, workspace=At())
    a.update(kw)
    (kv or paged()).tree_attention(s or seqs(), d or tree(), a.pop("query"), a.pop("out"),
                                   a.pop("heads"), **a)


def keep(layers=None, s=None, **kw):
    a = dict(path=At(), path_stride=40, counts=At())
    a.update(kw)
    nut.PagedLayers([paged(), paged()] if layers is None else layers).keep(
        s or seqs(), a["path"], a["path_stride"], a["counts"])


def copy(layers=None, copies=At(), count=5):
    nut.PagedLayers([paged(), paged()] if layers is None else layers).copy(copies, count)


def reorder(p=None, old=None, new=None, **kw):
    a = dict(parents=At(1 << 24), copies=At((1 << 24) + 4096), gain=1, workspace=At())
    a.update(kw)
    (p or pool()).reorder(old or table(), new or table(1 << 18), a.pop("parents"),
                          a.pop("copies"), **a)


def compact(p=None, t=None, **kw):
    a = dict(limit=5, copies=At(1 << 24), count=5, workspace=At())
    a.update(kw)
    (p or pool()).compact(t or table(), a.pop("limit"), a.pop("copies"), a.pop("count"), **a)


def select(old=None, new=None, **kw):
    a = dict(logits=At(), vocab=1000, parents=At(1 << 24), tokens=At((1 << 24) + 4096),
             workspace=At())
    a.update(kw)
    nut.beam_select(old or beams(), new or beams(1 << 22), a.pop("logits"), a.pop("vocab"),
                    a.pop("parents"), a.pop("tokens"), **a)


def gather(**kw):
    a = dict(source=At(), to=At(1 << 24), row_bytes=64, parents=At(), rows=3, sources=3)
    a.update(kw)
    nut.beam_gather(a.pop("source"), a.pop("to"), a.pop("row_bytes"), a.pop("parents"), **a)


CALLS = [build, accept, attention, keep, copy, reorder, compact, select, gather]


def refused(message, call, *a, **kw):
    with pytest.raises(nut.InvalidArgument, match=message):
        call(*a, **kw)


def reaches(call, *a, **kw):
    with pytest.raises(nut.DeviceError):
        call(*a, **kw)


@pytest.mark.parametrize("call", CALLS)
def test_valid_calls_reach_the_device(call):
    reaches(call)


@pytest.mark.parametrize("call", [build, accept, attention])
def test_trees(call):
    refused("invalid dimensions", call, tree(batch=0))
    refused("invalid dimensions", call, tree(most=0))
    refused("invalid dimensions", call, tree(total=1 << 31))
    refused("more than 1024 nodes", call, tree(most=1025))
    refused("without starts", call, tree(starts=None))
    refused("without starts", call, tree(starts=None, total=121))
    reaches(call, tree(starts=None, total=120))
    reaches(call, tree(most=1024, mask_stride=32))
    reaches(call, tree(total=0))
    if call is not accept:
        refused("null pointer", call, tree(mask=NONE))
        refused("masks shorter", call, tree(mask_stride=1))
        refused("masks shorter", call, tree(most=65, mask_stride=2))
        reaches(call, tree(most=64, mask_stride=2))
    if call is not attention:
        refused("null pointer", call, tree(parents=NONE))


def test_accept_arguments():
    for name in ("tokens", "chosen", "path", "counts"):
        refused("null pointer", accept, **{name: None})
    refused("null pointer", accept, s=seqs(lengths=NONE))
    refused("invalid batch", accept, s=seqs(batch=4))
    refused("paths shorter", accept, path_stride=39)
    refused("must not be the lengths", accept, new_lengths=At(8200))
    reaches(accept, new_lengths=At(8204), s=seqs(pages=None, stride=0))
    reaches(accept, new_lengths=None, last=None)


def test_attention_arguments():
    refused("multiple of the KV heads", attention, heads=7)
    refused("null pointer", attention, query=None)
    refused("null pointer", attention, out=None)
    refused("null pointer", attention, s=seqs(pages=NONE))
    refused("invalid batch", attention, s=seqs(batch=2))
    refused("page table shorter", attention, s=seqs(most=65))
    refused("16 bytes", attention, query=At(4100))
    refused("16 bytes", attention, out=At(4104))
    refused("16 bytes", attention, query_stride=514)
    refused("rows overlap", attention, query_stride=508)
    refused("unknown type", attention, kv=paged(dtype=3))
    for scale in (float("nan"), float("inf")):
        refused("scale is not finite", attention, scale=scale)
    big = dict(d=tree(most=1024, total=5000, mask_stride=32), s=seqs(stride=4096, most=65536))
    for args in (dict(d=tree(), s=seqs()), big):
        need = paged().tree_attention_workspace(args["s"], args["d"], 8)
        if need:
            refused("workspace too small", attention, workspace=At(nbytes=need - 1), **args)
            refused("workspace too small", attention, workspace=None, **args)
            refused("16-byte aligned", attention, workspace=At(4104), **args)
        reaches(attention, workspace=At(nbytes=need), **args)
    assert need > 0


def test_attention_launches_that_one_grid_does_not_cover():
    refused("more rows than one launch covers", paged(kv_heads=1).tree_attention_workspace,
            seqs(batch=65536, stride=64, most=1024), tree(batch=65536), 8)
    refused("more rows than one launch covers",
            paged(kv_heads=1 << 20, head_dim=8, page_size=1, pages=4).tree_attention_workspace,
            seqs(stride=64), tree(most=1024, mask_stride=32), 1 << 21)


@pytest.mark.parametrize("call", [keep, copy])
def test_layers(call):
    refused("no layers", call, [])
    for other in (dict(pages=11), dict(page_size=8), dict(kv_heads=1), dict(head_dim=32),
                  dict(dtype=nut.F16), dict(bounds=None), dict(strides=(4096, 2048, 72))):
        refused("layers of different shapes", call, [paged(), paged(**other)])
        # beyond the first launch's too, before anything runs
        refused("layers of different shapes", call, [paged()] * 69 + [paged(**other)])
    refused("null pointer", call, [paged(), paged(keys=NONE)])
    refused("16 bytes", call, [paged(), paged(values=At(4104))])
    reaches(call, [paged(keys=At(1 << 20)), paged(values=At(1 << 30))] * 50)
    many = [paged(kv_heads=65536, head_dim=8, pages=1)]
    refused("more rows than one launch covers", call, many)


def test_keep_arguments():
    refused("null pointer", keep, path=None)
    refused("null pointer", keep, counts=None)
    refused("paths shorter", keep, path_stride=0)
    refused("page table shorter", keep, s=seqs(most=65))


def test_copy_arguments():
    refused("null pointer", copy, copies=None)
    refused("invalid copies", copy, count=1 << 30)
    reaches(copy, copies=None, count=0)


@pytest.mark.parametrize("call", [reorder, compact])
def test_pools(call):
    refused("null pointer", call, pool(refs=None))
    for kw in (dict(pages=0), dict(pages=1 << 31), dict(page_size=0), dict(page_size=1 << 31)):
        refused("invalid dimensions", call, pool(**kw))
    for kw in (dict(pages=None), dict(lengths=None), dict(held=None)):
        refused("null pointer", call, None, table(**kw))
    for kw in (dict(stride=0), dict(batch=0), dict(stride=1 << 31), dict(batch=1 << 31)):
        refused("invalid table", call, None, table(**kw))
    refused("workspace too small", call, workspace=None)
    refused("workspace too small", call, workspace=At(nbytes=64))
    refused("16-byte aligned", call, workspace=At(4104))


def test_reorder_arguments():
    refused("null pointer", reorder, parents=None)
    refused("null pointer", reorder, copies=None)
    refused("invalid gain", reorder, gain=1 << 31)
    refused("invalid table", reorder, new=table(1 << 18, stride=0))
    base = 1 << 16  # the old table's 3 x 8 entries, three lengths and held pages
    for at in (base - 4, base + 92):
        refused("overlaps what is read", reorder, new=table(1 << 18, lengths=At(at)))
        refused("overlaps what is read", reorder, copies=At(at))
    reaches(reorder, new=table(1 << 18, lengths=At(base - 12)))
    reaches(reorder, new=table(1 << 18, lengths=At(base + 96)))
    refused("overlaps what is read", reorder, new=table(1 << 18, held=At(base + 4096 + 8)))
    refused("overlaps what is read", reorder, gains=At((1 << 18) + 92))
    refused("overlaps what is read", reorder, copies=At((1 << 24) - 4))
    refused("overlaps itself", reorder, copies=At((1 << 18) + 8192 - 32))
    refused("overlaps itself", reorder, new=table(1 << 18, held=At((1 << 18) + 4096)))
    need = pool().reorder_workspace(table(), table(1 << 18))
    refused("workspace too small", reorder, workspace=At(nbytes=need - 1))
    reaches(reorder, workspace=At(nbytes=need), gains=At())


def test_compact_arguments():
    refused("limit beyond", compact, limit=11)
    refused("null pointer", compact, copies=None)
    refused("invalid copies", compact, count=0)
    refused("invalid copies", compact, count=1 << 30)
    need = pool().compact_workspace(table())
    refused("workspace too small", compact, workspace=At(nbytes=need - 1))
    for limit in (0, 10):
        reaches(compact, limit=limit, workspace=At(nbytes=need))


def test_select_arguments():
    refused("null pointer", select, beams(scores=None))
    for kw in (dict(requests=0), dict(beams=0), dict(requests=1 << 31)):
        refused("invalid dimensions", select, beams(**kw))
    refused("more than 64 beams", select, beams(beams=65))
    refused("more than 64 beams", select, None, beams(1 << 22, beams=65))
    refused("different requests", select, None, beams(1 << 22, requests=3))
    refused("or neither", select, beams(lengths=None))
    refused("or neither", select, None, beams(1 << 22, ended=None))
    for vocab in (0, 262145):
        refused("vocabulary must be 1 to 262144", select, vocab=vocab)
    for name in ("logits", "parents", "tokens"):
        refused("null pointer", select, **{name: None})
    refused("unknown type", select, dtype=3)
    refused("rows overlap", select, row_stride=999)
    refused("misaligned logits", select, logits=At(4098))
    reaches(select, logits=At(4098), dtype=nut.F16)
    refused("misaligned logits", select, logits=At(4097), dtype=nut.BF16)
    refused("token out of range", select, eos=1000)
    refused("token out of range", select, eos=-2)
    for power in (float("nan"), float("inf"), 16.5, -17.0):
        refused("power must be -16 to 16", select, power=power)
    bare = dict(lengths=None, ended=None)
    refused("no lengths to rank by", select, beams(**bare), beams(1 << 22, **bare), power=0.5)
    reaches(select, beams(**bare), beams(1 << 22, **bare))
    base = 1 << 20
    for at in (base - 28, base + 28, base + 4096, base + 8192):
        refused("overlaps the old one", select, parents=At(at))
        refused("overlaps the old one", select, None, beams(1 << 22, scores=At(at)))
    reaches(select, parents=At(base + 32))
    need = nut.beam_select_workspace(beams(), beams(1 << 22), 1000)
    refused("workspace too small", select, workspace=At(nbytes=need - 1))
    refused("16-byte aligned", select, workspace=At(4104))
    reaches(select, workspace=At(nbytes=need), eos=999, power=-16.0, vocab=1000)


def test_gather_arguments():
    for name in ("source", "to", "parents"):
        refused("null pointer", gather, **{name: None})
    for kw in (dict(rows=0), dict(sources=0), dict(row_bytes=0), dict(rows=1 << 31),
               dict(row_bytes=1 << 40), dict(to_stride=1 << 40)):
        refused("invalid dimensions", gather, **kw)
    for kw in (dict(row_bytes=66), dict(source=At(4098)), dict(to=At((1 << 24) + 2)),
               dict(from_stride=70), dict(to_stride=66)):
        refused("multiples of 4 bytes", gather, **kw)
    refused("rows overlap", gather, to_stride=60)
    reaches(gather, to_stride=60, rows=1)
    reaches(gather, from_stride=4)  # sources may overlap one another
    for at in (4096 - 188, 4096, 4096 + 188):
        refused("rows overlap", gather, to=At(at))
    reaches(gather, to=At(4096 + 192))
    reaches(gather, to=At(4096 - 192))
    refused("more rows than one launch covers", gather, rows=1 << 30, to=At(1 << 44),
            row_bytes=4)


def test_workspaces_of_refused_calls():
    """(size_t)-1 through the C ABI, the refusal itself in Python."""
    L, kv, s = nut.lib(), paged(), seqs()
    wide = tree(most=1025)
    assert L.nut_paged_tree_attention_workspace(kv.ref, s.ref, wide.ref, 8) == C.c_size_t(-1).value
    assert b"more than 1024 nodes" in L.nut_last_error()
    refused("more than 1024 nodes", kv.tree_attention_workspace, s, wide, 8)
    refused("invalid table", pool().compact_workspace, table(batch=0))
    refused("invalid table", pool().reorder_workspace, table(), table(batch=0))
    refused("different requests", nut.beam_select_workspace, beams(), beams(requests=1), 10)


def test_null_views():
    L = nut.lib()
    assert L.nut_draft_mask(None, None, None) == 1
    assert L.nut_draft_accept(None, None, None, None, None, 1, None, None, None, None) == 1
    assert L.nut_paged_tree_attention(None, None, None, None, 0, 8, 1.0, None, None, None, 0,
                                      None) == 1
    assert L.nut_paged_keep(None, 1, None, None, 1, None, None) == 1
    assert L.nut_paged_copy(None, 1, None, 1, None) == 1
    assert L.nut_pages_reorder(None, None, None, None, None, 0, None, None, 0, None) == 1
    assert L.nut_pages_compact(None, None, 0, None, 1, None, 0, None) == 1
    assert L.nut_beam_select(None, None, None, 0, 0, 1, -1, 0.0, None, None, None, 0, None) == 1
    assert L.nut_beam_gather(None, 0, 1, None, 0, 1, 4, None, None, None) == 1
    assert L.nut_status_check(None) == 1
    assert L.nut_last_error() == b"paged cache: no status word"


@pytest.mark.parametrize("program", [["serving_index_test"], ["serving_api_test", "--cpu-only"]])
def test_cpp(program):
    """Masks, spans and parents as the kernels take them; the C++ host API's refusals."""
    build = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build")
    binary = os.path.join(build, program[0])
    assert os.path.exists(binary), "build first: make -C tests/cpp"
    r = subprocess.run([binary, *program[1:]], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr
