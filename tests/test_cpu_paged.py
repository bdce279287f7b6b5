"""What the paged KV cache's entry points refuse before anything is launched,
on a host without a GPU: each refusal's message, and that the arguments next to
it come through to the device (and fail there, loudly, where there is none)."""
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

KV = dict(pages=10, page_size=16, kv_heads=2, head_dim=64, dtype=nut.BF16)
SEQS = dict(table_stride=4, batch=3, max_length=64)


def paged(**kw):
    a = {**KV, **kw}
    return nut.PagedKV(a.pop("keys", At()), a.pop("values", At()), a.pop("pages"),
                       a.pop("page_size"), a.pop("kv_heads"), a.pop("head_dim"), a.pop("dtype"),
                       bounds=a.pop("bounds", At()), **a)


def seqs(**kw):
    a = {**SEQS, **kw}
    return nut.PagedBatch(a.get("pages", At()), a["table_stride"], a.get("lengths", At(8192)),
                          a["batch"], a["max_length"])


def history(stride=64, weights=At(), positions=At()):
    return nut.PagedHistory(weights, positions, stride)


def attention(kv=None, s=None, **kw):
    a = dict(query=At(), out=At(), heads=8, workspace=At())
    a.update(kw)
    (kv or paged()).attention(s or seqs(), a.pop("query"), a.pop("out"), a.pop("heads"), **a)


def select(kv=None, s=None, **kw):
    a = dict(query=At(), selected=At(), heads=8, top=3, workspace=At())
    a.update(kw)
    (kv or paged()).select(s or seqs(), a.pop("query"), a.pop("selected"), a.pop("heads"),
                           a.pop("top"), **a)


def evict(kv=None, s=None, **kw):
    a = dict(history=history(), new_lengths=At(), budget=32, workspace=At())
    a.update(kw)
    (kv or paged()).evict(s or seqs(), a.pop("history"), a.pop("new_lengths"), a.pop("budget"),
                          **a)


def append(kv=None, s=None, **kw):
    a = dict(keys=At(), values=At(), new_lengths=At())
    a.update(kw)
    (kv or paged()).append(s or seqs(), a.pop("keys"), a.pop("values"), a.pop("new_lengths"), **a)


def refused(message, call, *a, **kw):
    with pytest.raises(nut.InvalidArgument, match=message):
        call(*a, **kw)


@pytest.mark.parametrize("call", [attention, select, evict, append])
def test_valid_calls_reach_the_device(call):
    for kv in (paged(), paged(dtype=nut.F32, page_size=1, strides=(128, 64, 64)),
               paged(strides=(2048, 64, 128)),  # the heads of a row side by side
               paged(strides=(4096, 2048, 72)), paged(pages=1, strides=(0, 1024, 64))):
        with pytest.raises(nut.DeviceError):
            call(kv, seqs(table_stride=64))


@pytest.mark.parametrize("call", [attention, select, evict, append])
def test_views(call):
    none = At(None)
    refused("null pointer", call, paged(keys=none))
    refused("null pointer", call, paged(values=none))
    refused("unknown type", call, paged(dtype=3))
    refused("unknown type", call, paged(dtype=-1))
    for name in ("pages", "page_size", "kv_heads"):
        refused("invalid dimensions", call, paged(**{name: 0}))
        refused("invalid dimensions", call, paged(**{name: 1 << 31}))
    refused("invalid dimensions", call, paged(pages=(1 << 31) - 1, page_size=(1 << 31) - 1))
    for dim in (0, 4, 60, 264, 1 << 40):
        refused("head dim must be a multiple of 8 up to 256", call, paged(head_dim=dim))
    refused("16 bytes", call, paged(keys=At(4104)))
    refused("16 bytes", call, paged(values=At(4097)))
    refused("16 bytes", call, paged(bounds=At(4100)))
    refused("16 bytes", call, paged(strides=(4096, 2048, 68)))
    refused("16 bytes", call, paged(strides=(4100, 2048, 64)))
    refused("rows overlap", call, paged(strides=(4096, 2048, 56)))
    refused("rows overlap", call, paged(strides=(2040, 1024, 64)))
    refused("rows overlap", call, paged(strides=(0, 1024, 64)))
    refused("rows overlap", call, paged(strides=(2048, 56, 128)))
    refused("invalid dimensions", call, paged(strides=(1 << 62, 1024, 64)))
    refused("null pointer", call, None, seqs(pages=none))
    refused("null pointer", call, None, seqs(lengths=none))
    refused("invalid batch", call, None, seqs(batch=0))
    refused("invalid batch", call, None, seqs(max_length=0))
    refused("invalid batch", call, None, seqs(batch=1 << 31))
    refused("invalid batch", call, None, seqs(max_length=1 << 31, table_stride=1 << 28))
    refused("page table shorter", call, None, seqs(max_length=65))


def test_attention_arguments():
    refused("multiple of the KV heads", attention, heads=7)
    refused("multiple of the KV heads", attention, heads=0)
    refused("null pointer", attention, query=None)
    refused("null pointer", attention, out=None)
    refused("16 bytes", attention, query=At(4100))
    refused("16 bytes", attention, out=At(4104))
    refused("16 bytes", attention, query_stride=514)
    refused("rows overlap", attention, query_stride=508)
    for scale in (float("nan"), float("inf")):
        refused("scale is not finite", attention, scale=scale)
    refused("invalid selection", attention, selected=At())
    refused("invalid selection", attention, top=3)
    refused("invalid selection", attention, selected=At(), top=1 << 28)
    refused("no weights of a selection", attention, selected=At(), top=3, history=history())
    refused("history shorter", attention, history=history(63))
    refused("null history", attention, history=history(weights=None))
    refused("null history", attention, history=history(positions=None))
    need = paged().attention_workspace(seqs(), 8, weighted=True)
    refused("workspace too small", attention, history=history(), workspace=At(nbytes=need - 1))
    refused("workspace too small", attention, history=history(), workspace=None)
    refused("16-byte aligned", attention, history=history(), workspace=At(4100))
    with pytest.raises(nut.DeviceError):
        attention(history=history(), workspace=At(nbytes=need))
    with pytest.raises(nut.DeviceError):
        attention(query_stride=516, scale=0.0)


def test_select_arguments():
    refused("keeps no bounds", select, paged(bounds=None))
    refused("multiple of the KV heads", select, heads=3)
    refused("invalid selection", select, top=0)
    refused("first and last pages", select, first=2, last=2)
    refused("first and last pages", select, first=4, last=0)
    refused("first and last pages", select, first=(1 << 64) - 1, last=2)
    refused("null pointer", select, selected=None)
    refused("null pointer", select, query=None)
    need = paged().select_workspace(seqs(), 8, 3)
    refused("workspace too small", select, workspace=At(nbytes=need - 1))
    refused("16-byte aligned", select, workspace=At(4104))
    with pytest.raises(nut.DeviceError):
        select(workspace=At(nbytes=need), first=1, last=2)


def test_evict_arguments():
    refused("null history", evict, history=None)
    refused("history shorter", evict, history=history(1))
    refused("invalid budget", evict, budget=0)
    refused("first and last rows", evict, first=16, last=17)
    refused("first and last rows", evict, first=0, last=(1 << 64) - 1)
    refused("null pointer", evict, new_lengths=None)
    refused("must not be the lengths", evict, new_lengths=At(8192))
    need = paged().evict_workspace(seqs(), 32)
    refused("workspace too small", evict, workspace=At(nbytes=need - 1))
    refused("16-byte aligned", evict, workspace=At(4104))
    with pytest.raises(nut.DeviceError):
        evict(workspace=At(nbytes=need), first=16, last=16)


def test_append_arguments():
    refused("null pointer", append, keys=At(None))
    refused("must not be the lengths", append, new_lengths=At(8192))
    refused("one row a sequence", append, max_new=2)
    refused("one row a sequence", append, keys=At(nbytes=4 * 2 * 64 * 3 - 1))
    refused("invalid row count", append, max_new=0, starts=At())
    refused("16 bytes", append, keys=At(4100))
    refused("16 bytes", append, values=At(4100))
    refused("16 bytes", append, row_stride=386, head_stride=64)
    refused("16 bytes", append, row_stride=384, head_stride=65)
    refused("invalid strides", append, row_stride=1 << 31, head_stride=64, starts=At())
    refused("history shorter", append, history=history(1))
    with pytest.raises(nut.DeviceError):
        append(keys=At(nbytes=4 * 2 * 64 * 3), new_lengths=None)


def test_append_strides():
    """Each stride of 0 is that of packed rows, whatever the other one is;
    source rows or heads that overlap are refused."""
    # three sequences' rows of two heads of 64, alone and among others
    for strides in (dict(row_stride=384), dict(head_stride=64), dict(row_stride=128),
                    dict(row_stride=64, head_stride=192), dict(row_stride=384, head_stride=128),
                    dict()):
        with pytest.raises(nut.DeviceError):
            append(keys=At(nbytes=4 * (2 * (strides.get("row_stride") or 128) +
                                       (strides.get("head_stride") or 64) + 64)), **strides)
    for strides in (dict(head_stride=192), dict(head_stride=128), dict(row_stride=64),
                    dict(row_stride=124), dict(row_stride=192, head_stride=192),
                    dict(row_stride=384, head_stride=32)):
        refused("rows overlap", append, **strides)
    # heads before rows: as many rows as there are before the next head
    refused("one row a sequence", append, row_stride=64, head_stride=128)
    for head_stride in (192, 200, 6400):
        with pytest.raises(nut.DeviceError):
            append(row_stride=64, head_stride=head_stride)
    # one row, or one head, has nothing to overlap with
    one = seqs(batch=1)
    with pytest.raises(nut.DeviceError):
        append(s=one, keys=At(nbytes=4 * (192 + 64)), head_stride=192)
    with pytest.raises(nut.DeviceError):
        append(paged(kv_heads=1), head_stride=4)


def test_new_lengths_that_overlap_an_input():
    """The lengths are at 8192: three integers."""
    for call in (append, evict):
        for at in (8184, 8188, 8196, 8200):
            refused("must not be the lengths", call, new_lengths=At(at))
        for at in (8180, 8204):
            with pytest.raises(nut.DeviceError):
                call(new_lengths=At(at))
    for at in (12280, 12288, 12300):  # four starts
        refused("starts or first positions", append, starts=At(12288), new_lengths=At(at))
    for at in (12280, 12288, 12296):
        refused("starts or first positions", append, first_positions=At(12288),
                new_lengths=At(at))
    with pytest.raises(nut.DeviceError):
        append(starts=At(12288), first_positions=At(12304), new_lengths=At(12276))


def test_append_from_a_cache_refuses():
    L, kv, s = nut.lib(), paged(), seqs(batch=1)
    assert L.nut_paged_append_cache(kv.ref, s.ref, None, 0, 0, 1, None, None, None, None) == 1
    assert L.nut_last_error() == b"kv cache: null cache"


def test_workspaces_of_refused_calls():
    """(size_t)-1 through the C ABI, the refusal itself in Python."""
    L = nut.lib()
    kv, s = paged(), seqs()
    assert L.nut_paged_attention_workspace(kv.ref, s.ref, 7, 0, 0) == C.c_size_t(-1).value
    assert b"multiple of the KV heads" in L.nut_last_error()
    refused("multiple of the KV heads", kv.attention_workspace, s, 7)
    refused("no weights of a selection", kv.attention_workspace, s, 8, top=2, weighted=True)
    refused("invalid selection", kv.select_workspace, s, 8, 0)
    refused("invalid budget", kv.evict_workspace, s, 0)


def test_eviction_workspace_grows_with_the_rows_that_can_move():
    """One that keeps all but one row, or every row, of 64 needs little."""
    sizes = [paged().evict_workspace(seqs(), budget) for budget in (63, 64, 1 << 30)]
    assert max(sizes) <= 768 and paged().evict_workspace(seqs(), 32) > 768


def test_check_needs_a_status_word():
    refused("no status word", paged().check)


def test_null_views():
    L = nut.lib()
    assert L.nut_paged_check(None) == 1
    assert L.nut_paged_select(None, None, None, 0, 8, 3, 0, 0, None, None, 0, None) == 1
    assert L.nut_paged_evict(None, None, None, 8, 0, 0, None, None, 0, None) == 1
    assert L.nut_paged_append(None, None, None, None, 0, 0, 0, None, 1, None, None, None, None) == 1
    assert L.nut_paged_attention(None, None, None, 0, 8, 1.0, None, 0, None, None, None, None, 0,
                                 None) == 1


@pytest.mark.parametrize("program", [["paged_index_test"], ["paged_api_test", "--cpu-only"]])
def test_cpp(program):
    """Pages, lengths and counts as the kernels judge them, and where rows
    go; the C++ host API's refusals."""
    build = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build")
    binary = os.path.join(build, program[0])
    assert os.path.exists(binary), "build first: make -C tests/cpp"
    r = subprocess.run([binary, *program[1:]], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr


def test_launches_that_one_grid_does_not_cover():
    big = dict(kv_heads=1 << 20, head_dim=8, page_size=1, pages=4)
    refused("more rows than one launch covers", paged(**big).attention_workspace,
            seqs(table_stride=64, batch=8), 1 << 20)
    refused("more rows than one launch covers", paged(**big).select_workspace,
            seqs(table_stride=64, batch=128), 1 << 20, 3)
    refused("more rows than one launch covers", paged(**big).evict_workspace,
            seqs(table_stride=64, batch=128), 8)
    refused("more rows than one launch covers", paged(kv_heads=1).attention_workspace,
            seqs(table_stride=64, batch=65536), 8)


def test_second_launches_that_one_grid_does_not_cover():
    """The launches behind a call's first are looked at with it, so that nothing
    runs of a call that is refused, and its workspace is refused too."""
    # 2^21 heads whose lists of 1,000 to 3,000 moved rows take 4 to 12 workgroups each
    many = dict(kv_heads=64, head_dim=8, page_size=64, pages=4)
    s = dict(table_stride=100, batch=1 << 15, max_length=6000)
    paged(**many).evict_workspace(seqs(**s), 1000)
    refused("more rows than one launch covers", paged(**many).evict_workspace, seqs(**s), 3000)
    refused("more rows than one launch covers", evict, paged(**many), seqs(**s), budget=3000,
            history=history(6000), workspace=At(nbytes=1 << 60), new_lengths=At(1 << 40))
    # 2^26 query heads of two runs each, joined by a wave a head
    wide = dict(kv_heads=1, head_dim=8, page_size=64, pages=4)
    s = dict(table_stride=64, batch=1 << 15, max_length=2049)
    paged(**wide).attention_workspace(seqs(**s), 1 << 10)
    refused("more rows than one launch covers", paged(**wide).attention_workspace, seqs(**s),
            1 << 11)
    refused("more rows than one launch covers", attention, paged(**wide), seqs(**s), heads=1 << 11,
            workspace=At(nbytes=1 << 60))
