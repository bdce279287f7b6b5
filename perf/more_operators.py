"""Performance cases of what serves several continuations of a text from one
paged KV cache: attention of a tree of drafted tokens, its verification (mask,
accepted path, rows kept), forked and compacted page tables with the copies
they ask for, and beam search's selection.

``run`` computes a case with elementary torch operations in 32 bits (64 where
whole numbers hang on them), or, with ``own``, through the framework's entry
points. The shapes are the repository's synthetic workloads (the TinyLlama
and Llama-2-7B attention shapes, layers and vocabulary, the small test shapes)
and generic odd ones.

Inputs come from the seed alone; lengths, node counts and which continuations
live on come from the case, so that ``work`` can count. Pages lie in no order.
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

SHAPES = {  # heads, KV heads, head dim, layers
    "tiny": (4, 2, 16, 2),
    "step_gqa2": (4, 2, 64, 2),
    "step_gqa4": (8, 2, 64, 2),
    "step_mha128": (2, 2, 128, 2),
    "tinyllama": (32, 4, 64, 22),
    "llama7b": (32, 32, 128, 32),
    "odd": (24, 3, 80, 5),  # a generic width that no power of two divides into
}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EOS = 1


def listed():
    return [
        # one chat with a short context and a small tree: where latency counts
        dict(name="tree_chat", kind="tree", shape="tinyllama", type="f32", batch=1, low=211,
             high=211, nodes=16, page=16, order="head", idle=0),
        # an ordinary serving batch, ragged trees, one idle slot
        dict(name="tree_batch", kind="tree", shape="tinyllama", type="bf16", batch=16, low=1,
             high=2048, nodes=64, page=16, order="head", idle=1),
        # long documents on the 7B widths, one KV head per query head
        dict(name="tree_long", kind="tree", shape="llama7b", type="f16", batch=4, low=24000,
             high=32768, nodes=64, page=64, order="head", idle=0),
        # odd sizes: 80 dims, pages of 24 rows, the heads of a row side by side, wide trees
        dict(name="tree_odd", kind="tree", shape="odd", type="f32", batch=7, low=1, high=5001,
             nodes=203, page=24, order="slot", idle=0),
        # a decode step's verification: masks, accepted paths, their rows in every layer
        dict(name="verify_step", kind="verify", shape="tinyllama", type="bf16", batch=16, low=1,
             high=2048, nodes=64, page=16, order="head", idle=1),
        # the same for many short texts on the 7B widths
        dict(name="verify_wide", kind="verify", shape="llama7b", type="f16", batch=32, low=1,
             high=64, nodes=27, page=64, order="head", idle=0),
        # a step of beam search: the table follows the beams that live on, pages that part
        # are copied in every layer
        dict(name="fork_beams", kind="fork", shape="tinyllama", type="bf16", batch=32, beams=4,
             keep=4, low=100, high=1500, page=16, order="head"),
        # several samples of each prompt: one sequence becomes eight
        dict(name="fork_samples", kind="fork", shape="llama7b", type="f16", batch=8, beams=1,
             keep=8, low=60, high=500, page=64, order="head"),
        # the smallest: two beams of one text on a small shape
        dict(name="compact_small", kind="compact", shape="step_gqa4", type="f32", pages=64,
             batch=3, page=16, order="head", limit=36),
        # a server gives the upper part of its cache back: moved pages in every layer
        dict(name="compact_pool", kind="compact", shape="tinyllama", type="bf16", pages=4096,
             batch=48, page=16, order="head", limit=2500),
        # beam search on one text
        dict(name="beam_one", kind="beam", type="f32", batch=1, beams=4, keep=4, vocab=32000,
             power=0.0, ended=0, first=False, text=64),
        # a full batch, a large odd vocabulary in 16 bits, scores by length, ended beams
        dict(name="beam_batch", kind="beam", type="f16", batch=64, beams=8, keep=8,
             vocab=100003, power=0.7, ended=2, first=False, text=1000),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "verify", "fork", "fork", "compact", "beam",
                       "beam"])
    if kind == "beam":
        beams = _log_int(rng, 1, 16)
        case = dict(kind=kind, type=rng.choice(["f32", "f32", "f16", "bf16"]),
                    batch=_log_int(rng, 1, 64), beams=beams,
                    keep=rng.choice([beams, _log_int(rng, 1, 32)]),
                    power=rng.choice([0.0, 0.0, 0.6, 1.0]), first=rng.random() < 0.2,
                    text=_log_int(rng, 1, 2000))
        most = int(5e7 / case["batch"] / beams)
        case["vocab"] = _log_int(rng, 50, min(200000, most))
        case["keep"] = min(case["keep"], case["vocab"])
        case["ended"] = 0 if case["first"] else rng.choice([0, beams // 4])
        return case
    shape = rng.choice(["tiny", "step_gqa2", "step_gqa4", "step_mha128", "tinyllama", "tinyllama",
                        "llama7b", "llama7b", "odd"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    heads, kv, dim, layers = SHAPES[shape]
    case = dict(kind=kind, shape=shape, type=dtype, page=rng.choice([8, 16, 16, 24, 32, 64, 128]),
                order=rng.choice(["head", "head", "slot"]))
    row = 2 * kv * dim * (4 if dtype == "f32" else 2)
    if kind == "compact":
        most = int(1.5e9 / (row * layers * case["page"]))
        case["pages"] = max(9, min(8192, _log_int(rng, 9, most)))
        case["batch"] = rng.randint(1, max(1, case["pages"] // 8))
        case["limit"] = rng.randint(case["pages"] // 2, case["pages"] - 1)
        return case
    if kind == "fork":
        case["batch"], case["beams"] = _log_int(rng, 1, 32), _log_int(rng, 1, 8)
        case["keep"] = rng.choice([case["beams"], _log_int(rng, 1, 8)])
        each = max(case["beams"], case["keep"]) * 2
        most = int(1.5e9 / (row * layers * case["batch"] * each))
        case["page"] = min(case["page"], max(8, most // 4 // 8 * 8))
        case["high"] = _log_int(rng, 1, min(8000, max(2, most - 2 * case["page"])))
        case["low"] = rng.randint(1, case["high"])
        return case
    case["batch"], case["nodes"] = _log_int(rng, 1, 64), _log_int(rng, 1, 256)
    if kind == "verify":
        case["nodes"] = min(case["nodes"], 128)
        least = row * layers * (case["nodes"] + 2 * case["page"])
        case["batch"] = max(1, min(case["batch"], 32, int(1.5e9 / least)))
        most = int(1.5e9 / (row * layers * case["batch"])) - case["nodes"] - case["page"]
        case["high"] = _log_int(rng, 1, min(4000, max(2, most)))
    else:
        most = min(1.0e9 / row / case["batch"], 1.0e11 / (4 * heads * dim * case["nodes"]) /
                   case["batch"], 2.5e8 / (heads * case["nodes"]) / case["batch"])
        case["high"] = _log_int(rng, 1, min(32768, max(2, int(most) - case["nodes"])))
    case["low"] = rng.randint(1, case["high"])
    case["idle"] = rng.choice([0, 0, case["batch"] // 8])
    return case


# ------------------------------------------------------------------ inputs --

def _spread(i, low, high):
    return high if i == 0 else low + int((i * 0.6180339887) % 1.0 * (high - low + 1))


def _lengths(case):
    """Rows of each sequence: spread evenly over the case's range, idle ones at the end."""
    n = case["batch"] - case.get("idle", 0)
    return [_spread(i, case["low"], case["high"]) for i in range(n)] + [0] * case.get("idle", 0)


def _counts(case):
    """Drafted tokens of each sequence."""
    n, most = case["batch"] - case["idle"], case["nodes"]
    return [most if i == 0 else 1 + int((i * 0.7548776662) % 1.0 * most) for i in range(n)] + \
        [0] * case["idle"]


def _parents(case):
    """The sequences that the kept continuations go on with: of each request's beams, some
    live on once, some more often, some not at all."""
    beams, keep = case["beams"], case["keep"]
    return [r * beams + int(((r * 7 + k) * 0.5698402910) % 1.0 * beams)
            for r in range(case["batch"]) for k in range(keep)]


def _gen(seed, stream):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + stream)


def _normal(seed, stream, *shape, sigma=1.0):
    return torch.randn(*shape, generator=_gen(seed, stream), device="cuda") * sigma


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pools(case, layers, pages, seed, stream):
    """Rows of every page, [layers, pages, kv_heads, page, dim] whichever way they lie."""
    _, kv, dim, _ = SHAPES[case["shape"]]
    rows = torch.empty(layers, pages, kv, case["page"], dim, device="cuda",
                       dtype=DTYPES[case["type"]])
    rows.normal_(0.0, 1.0, generator=_gen(seed, stream))
    if case["order"] == "slot":
        return rows.transpose(2, 3).contiguous().transpose(2, 3)
    return rows


def _bounds(keys):
    return torch.stack((keys.amin(3), keys.amax(3)), 3)


def _tree(case, seed):
    """Trees whose nodes have a few children each: a node's parent stands at a third to
    five sixths of its own place."""
    counts, most = _counts(case), case["nodes"]
    starts = [sum(counts[:i]) for i in range(case["batch"] + 1)]
    s = dict(starts=_ints(starts), total=starts[-1], most=most, words=-(-most // 32))
    at = torch.cat([torch.arange(c, device="cuda") for c in counts])
    u = torch.rand(s["total"], generator=_gen(seed, 60), device="cuda")
    parents = ((at - 1) * (0.33 + 0.5 * u)).long()
    s["parents"] = torch.where(at == 0, -1, parents).int()
    return s


def prepare(case, seed):
    kind = case["kind"]
    s = {"tree": _prepare_tree, "verify": _prepare_tree, "fork": _prepare_fork,
         "compact": _prepare_compact, "beam": _prepare_beam}[kind](case, seed)
    s.update(kind=kind, case=case)
    if own:
        _handles(s)
    return s


def _prepare_tree(case, seed):
    heads, kv, dim, layers = SHAPES[case["shape"]]
    ps, batch = case["page"], case["batch"]
    lengths, counts = _lengths(case), _counts(case)
    longest = max(n + m for n, m in zip(lengths, counts))
    width = -(-longest // ps)
    pages = batch * width + 3
    layers = 1 if case["kind"] == "tree" else layers
    order = torch.randperm(pages, generator=_gen(seed, 1), device="cuda")
    s = dict(_tree(case, seed), layers=layers, pages=pages, width=width, longest=longest,
             lengths=_ints(lengths), scale=dim ** -0.5,
             table=order[:batch * width].reshape(batch, width).int().contiguous(),
             keys=_pools(case, layers, pages, seed, 10),
             values=_pools(case, layers, pages, seed, 20))
    total, most = s["total"], s["most"]
    if case["kind"] == "tree":
        s["mask"] = _bits(_ancestors(s), s)
        s["query"] = _normal(seed, 30, total, heads, dim, sigma=1.5)
        s["out"] = torch.empty(total, heads, dim, device="cuda")
        s["lse"] = torch.empty(total, heads, device="cuda")
        return s
    s["bounds"] = _bounds(s["keys"])
    s["tokens"] = torch.randint(0, 3, (total,), generator=_gen(seed, 61), device="cuda").int()
    s["chosen"] = torch.randint(0, 3, (total,), generator=_gen(seed, 62), device="cuda").int()
    s["mask"] = torch.zeros(total, s["words"], dtype=torch.int32, device="cuda")
    s["depths"] = torch.zeros(total, dtype=torch.int32, device="cuda")
    s["path"] = torch.zeros(batch, most, dtype=torch.int32, device="cuda")
    for name in ("counts", "last", "new_lengths"):
        s[name] = torch.zeros(batch, dtype=torch.int32, device="cuda")
    return s


def _prepare_fork(case, seed):
    """Each request's beams share the pages of its prompt and hold the others alone."""
    _, _, _, layers = SHAPES[case["shape"]]
    ps, beams, keep = case["page"], case["beams"], case["keep"]
    lengths = _lengths(case)
    need = [-(-n // ps) for n in lengths]
    shared = [int(0.7 * n) // ps for n in lengths]
    spare = case["batch"] * keep * 2 + 5
    pages = sum(c + beams * (n - c) for c, n in zip(shared, need)) + spare
    width = max(need) + 2
    order = torch.randperm(pages, generator=_gen(seed, 1), device="cuda").int()
    table = torch.full((case["batch"] * beams, width), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    at = 0
    for r, (c, n) in enumerate(zip(shared, need)):
        rows = slice(r * beams, (r + 1) * beams)
        table[rows, :c] = order[at:at + c]
        refs[order[at:at + c].long()] = beams
        at += c
        if n > c:
            mine = order[at:at + beams * (n - c)]
            table[rows, c:n] = mine.reshape(beams, n - c)
            refs[mine.long()] = 1
            at += beams * (n - c)
    kept = case["batch"] * keep
    s = dict(layers=layers, pages=pages, width=width, batch=case["batch"] * beams, kept=kept,
             keys=_pools(case, layers, pages, seed, 10),
             values=_pools(case, layers, pages, seed, 20), table=table, refs=refs,
             left=refs.clone(), lengths=_ints([n for n in lengths for _ in range(beams)]),
             held=_ints([n for n in need for _ in range(beams)]), parents=_ints(_parents(case)),
             new_table=torch.full((kept, width), -1, dtype=torch.int32, device="cuda"),
             new_lengths=torch.zeros(kept, dtype=torch.int32, device="cuda"),
             new_held=torch.zeros(kept, dtype=torch.int32, device="cuda"),
             copies=torch.zeros(kept, 3, dtype=torch.int32, device="cuda"))
    s["bounds"] = _bounds(s["keys"])
    return s


def _prepare_compact(case, seed):
    """About half of the pages are held; every third sequence shares its first page with
    the one before."""
    _, _, _, layers = SHAPES[case["shape"]]
    pages, batch = case["pages"], case["batch"]
    order = torch.randperm(pages, generator=_gen(seed, 1), device="cuda").int()
    each = [_spread(i, 1, max(1, pages // (2 * batch))) for i in range(batch)]
    width = max(each) + 1
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(each):
        mine = order[at:at + n]
        table[b, :n] = mine
        if b % 3 == 2:
            table[b, 0] = table[b - 1, 0]
        refs.index_add_(0, table[b, :n].long(), torch.ones_like(mine))
        at += n
    return dict(layers=layers, pages=pages, width=width, batch=batch, table=table, refs=refs,
                left=refs.clone(), left_table=table.clone(), held=_ints(each),
                lengths=_ints([n * case["page"] for n in each]),
                copies=torch.zeros(pages - case["limit"], 3, dtype=torch.int32, device="cuda"),
                keys=_pools(case, layers, pages, seed, 10),
                values=_pools(case, layers, pages, seed, 20))


def _prepare_beam(case, seed):
    batch, beams, keep = case["batch"], case["beams"], case["keep"]
    logits = _normal(seed, 70, batch * beams, case["vocab"], sigma=3.0).to(DTYPES[case["type"]])
    scores = -torch.rand(batch, beams, generator=_gen(seed, 71), device="cuda") * 4 - 8
    ended = torch.zeros(batch, beams, dtype=torch.int32, device="cuda")
    ended[:, beams - case["ended"]:] = 1
    lengths = torch.randint(5, 40, (batch, beams), generator=_gen(seed, 72), device="cuda").int()
    if case["first"]:  # after the prompt: one beam, the others are none yet
        scores[:, 1:] = -math.inf
        scores[:, 0] = 0.0
        lengths.zero_()
    empty = lambda *shape, dtype=torch.int32: torch.zeros(*shape, dtype=dtype,  # noqa: E731
                                                          device="cuda")
    return dict(logits=logits, scores=scores, ended=ended, lengths=lengths,
                text=torch.randint(0, 32000, (batch * beams, case["text"]),
                                   generator=_gen(seed, 73), device="cuda").int(),
                new_text=empty(batch * keep, case["text"]), parents=empty(batch, keep),
                tokens=empty(batch, keep), new_scores=empty(batch, keep, dtype=torch.float32),
                new_lengths=empty(batch, keep), new_ended=empty(batch, keep))


# ------------------------------------------------- the framework's kernels --

class _Buffer:
    """A torch tensor as the device buffer that the entry points take."""

    def __init__(self, tensor):
        self.tensor = tensor
        self.nbytes = tensor.numel() * tensor.element_size()
        self.ptr = ctypes.c_void_p(tensor.data_ptr())


def _space(need):
    return _Buffer(torch.empty(max(1, need), dtype=torch.uint8, device="cuda"))


def _handles(s):
    """The views of the cache, its table and its sequences, and the workspace, that a
    program keeps."""
    import nutllm_amd as nut

    case, kind = s["case"], s["kind"]
    b = s["b"] = {k: _Buffer(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
    types = {"f32": nut.F32, "f16": nut.F16, "bf16": nut.BF16}
    if kind == "beam":
        s["from"] = nut.BeamState(b["scores"], case["batch"], case["beams"],
                                  lengths=b["lengths"], ended=b["ended"])
        s["to"] = nut.BeamState(b["new_scores"], case["batch"], case["keep"],
                                lengths=b["new_lengths"], ended=b["new_ended"])
        s["type"] = types[case["type"]]
        s["space"] = _space(nut.beam_select_workspace(s["from"], s["to"], case["vocab"]))
        return
    _, kv, dim, _ = SHAPES[case["shape"]]
    views = [nut.PagedKV(_Buffer(s["keys"][i]), _Buffer(s["values"][i]), s["pages"],
                         case["page"], kv, dim, types[case["type"]],
                         strides=s["keys"].stride()[1:4],
                         bounds=_Buffer(s["bounds"][i]) if "bounds" in s else None)
             for i in range(s["layers"])]
    s["paged"], s["all"] = views[0], nut.PagedLayers(views)
    if kind in ("tree", "verify"):
        s["seqs"] = nut.PagedBatch(b["table"], s["width"], b["lengths"], case["batch"],
                                   s["longest"])
        s["draft"] = nut.DraftTree(b.get("parents"), b["mask"], s["most"], s["total"],
                                   case["batch"], starts=b["starts"])
        if kind == "tree":
            s["space"] = _space(s["paged"].tree_attention_workspace(
                s["seqs"], s["draft"], SHAPES[case["shape"]][0]))
        return
    s["pool"] = nut.PagePool(b["refs"], s["pages"], case["page"])
    s["now"] = nut.PageTable(b["table"], s["width"], b["lengths"], b["held"], s["batch"])
    if kind == "fork":
        s["next"] = nut.PageTable(b["new_table"], s["width"], b["new_lengths"], b["new_held"],
                                  s["kept"])
        s["space"] = _space(s["pool"].reorder_workspace(s["now"], s["next"]))
    else:
        s["space"] = _space(s["pool"].compact_workspace(s["now"]))


def _own(s):
    case, b, kind = s["case"], s["b"], s["kind"]
    if kind == "tree":
        s["paged"].tree_attention(s["seqs"], s["draft"], b["query"], b["out"],
                                  SHAPES[case["shape"]][0], scale=s["scale"], lse=b["lse"],
                                  workspace=s["space"])
    elif kind == "verify":
        s["draft"].build(depths=b["depths"])
        s["draft"].accept(s["seqs"], b["tokens"], b["chosen"], b["path"], b["counts"],
                          last=b["last"], new_lengths=b["new_lengths"])
        s["all"].keep(s["seqs"], b["path"], s["most"], b["counts"])
    elif kind == "fork":
        s["refs"].copy_(s["left"])  # what the step before left
        s["pool"].reorder(s["now"], s["next"], b["parents"], b["copies"], gain=1,
                          workspace=s["space"])
        s["all"].copy(b["copies"], s["kept"])
    elif kind == "compact":
        s["refs"].copy_(s["left"])
        s["table"].copy_(s["left_table"])
        s["pool"].compact(s["now"], case["limit"], b["copies"], s["copies"].shape[0],
                          workspace=s["space"])
        s["all"].copy(b["copies"], s["copies"].shape[0])
    else:
        import nutllm_amd as nut

        nut.beam_select(s["from"], s["to"], b["logits"], case["vocab"], b["parents"],
                        b["tokens"], dtype=s["type"], eos=EOS, power=case["power"],
                        workspace=s["space"])
        nut.beam_gather(b["text"], b["new_text"], 4 * case["text"], b["parents"],
                        rows=case["batch"] * case["keep"], sources=case["batch"] * case["beams"])
    return _state(s)


# ------------------------------------------------------------- plain forms --

OUTPUTS = {
    "tree": ("out", "lse"),
    "verify": ("mask", "depths", "path", "counts", "last", "new_lengths", "keys", "values",
               "bounds"),
    "fork": ("refs", "new_table", "new_lengths", "new_held", "copies", "keys", "values",
             "bounds"),
    "compact": ("refs", "table", "copies", "keys", "values"),
    "beam": ("parents", "tokens", "new_scores", "new_lengths", "new_ended", "new_text"),
}


def _state(s):
    return {k: s[k] for k in OUTPUTS[s["kind"]]}


def _padded(s):
    """Rows of [total] that nodes of [batch, most] lie in, and which of these there are."""
    at = torch.arange(s["most"], device="cuda")
    starts = s["starts"].long()
    inside = at < starts.diff()[:, None]
    return torch.where(inside, starts[:-1, None] + at, 0), inside


def _ancestors(s):
    """[batch, most, most]: whether node i sees node j, its ancestor or itself."""
    row, inside = _padded(s)
    parents = s["parents"].long()[row].masked_fill(~inside, -1)
    at = torch.arange(s["most"], device="cuda")
    step = ((parents[..., None] == at) | (at[:, None] == at)).float()
    for _ in range(s["most"].bit_length()):  # paths twice as long each time
        step = torch.matmul(step, step).clamp(max=1.0)
    return (step > 0) & inside[..., None] & inside[:, None]


def _bits(sees, s):
    """Rows of [batch, most, most] truth values as words, for the nodes that there are."""
    _, inside = _padded(s)
    wide = torch.nn.functional.pad(sees[inside], (0, s["words"] * 32 - s["most"]))
    weight = 2 ** torch.arange(32, device="cuda")
    words = (wide.reshape(s["total"], s["words"], 32) * weight).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()


def _rows(pool, table):
    """[batch, kv, rows, dim] of the pages that a table names, in 32 bits."""
    b, w = table.shape
    got = pool[table.long()].transpose(1, 2)  # [b, kv, w, page, dim]
    return got.reshape(b, got.shape[1], -1, got.shape[-1]).float()


def _attend(s):
    heads, kv, dim, _ = SHAPES[s["case"]["shape"]]
    batch, most = s["case"]["batch"], s["most"]
    row, inside = _padded(s)
    bits = s["mask"][row][..., None] >> torch.arange(32, device="cuda") & 1
    sees = bits.reshape(batch, most, -1)[..., :most].bool()  # [batch, node, node]
    k, v = _rows(s["keys"][0], s["table"]), _rows(s["values"][0], s["table"])
    at = torch.arange(k.shape[2], device="cuda")
    j = at - s["lengths"].long()[:, None]  # of [batch, rows]: which node's row it is
    drafted = (j >= 0) & (j < s["starts"].diff()[:, None])
    seen = sees.gather(2, j.clamp(0, most - 1)[:, None].expand(-1, most, -1))
    seen = torch.where(drafted[:, None], seen, (j < 0)[:, None])
    q = (s["query"][row] * s["scale"]).reshape(batch, most, kv, heads // kv, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(batch, kv, -1, dim)
    hidden = ~seen.repeat_interleave(heads // kv, 1)[:, None]
    score = torch.matmul(q, k.transpose(-1, -2)).masked_fill_(hidden, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = top.masked_fill(top == -math.inf, 0.0)
    p = torch.exp(score.sub_(top))
    z = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / z.masked_fill(z == 0.0, 1.0)
    back = lambda x: x.reshape(batch, kv, most, heads // kv, -1).transpose(1, 2)[inside]  # noqa
    s["out"].copy_(back(out).reshape(-1, heads, dim))
    s["lse"].copy_(back(top + z.log()).reshape(-1, heads))
    return _state(s)


def _verify(s):
    batch, most, ps = s["case"]["batch"], s["most"], s["case"]["page"]
    row, inside = _padded(s)
    sees = _ancestors(s)
    s["mask"].copy_(_bits(sees, s))
    s["depths"].copy_(sees.sum(-1)[inside] - 1)
    # a node goes on with its parent's choice if its token says so and no sibling before it does
    at = torch.arange(most, device="cuda")
    parents = s["parents"].long()[row].masked_fill(~inside, -1)
    tokens = s["tokens"][row]
    match = (parents >= 0) & (tokens == s["chosen"][row].gather(1, parents.clamp(min=0)))
    twin = match[:, None] & (parents[..., None] == parents[:, None]) & (at < at[:, None])
    ok = (match & ~twin.any(-1)) | ((at == 0) & inside)
    kept = inside & ~(sees & ~ok[:, None]).any(-1)
    counts = kept.sum(-1)
    order = (~kept).to(torch.int8).sort(dim=-1, stable=True)[1]  # kept nodes first
    there = at < counts[:, None]
    s["path"].copy_(torch.where(there, order, s["path"].long()))
    s["counts"].copy_(counts)
    tip = row.gather(1, s["path"].long().gather(1, (counts - 1).clamp(min=0)[:, None]))[:, 0]
    s["last"].copy_(torch.where(counts > 0, s["chosen"][tip], s["last"]))
    torch.add(s["lengths"], s["counts"], out=s["new_lengths"])
    # rows of the path, behind the sequence's rows; where there is none a row moves to itself
    seq = torch.arange(batch, device="cuda")[:, None]
    spot = s["lengths"].long()[:, None] + torch.where(there, s["path"].long(), 0)
    to = s["lengths"].long()[:, None] + torch.where(there, at, 0)
    live = torch.nonzero(there & (spot != to))  # what stays where it is is not moved
    seq, k = live[:, 0], live[:, 1]
    spot, to = spot[seq, k], to[seq, k]
    table = s["table"].long()
    source, page = table[seq, spot // ps], table[seq, to // ps]
    for pool in (s["keys"], s["values"]):
        pool[:, page, :, to % ps] = pool[:, source, :, spot % ps]
    moved = s["keys"][:, page, :, to % ps].transpose(0, 1).float()
    lo, hi = (x.float() for x in s["bounds"].unbind(3))
    lo.index_reduce_(1, page, moved, "amin")
    hi.index_reduce_(1, page, moved, "amax")
    s["bounds"].copy_(torch.stack((lo, hi), 3))
    return _state(s)


def _copy(s, source, to, rows):
    """Rows below `rows` of pages `source` into pages `to`, in every layer."""
    slot = torch.arange(s["case"]["page"], device="cuda") < rows[:, None]
    for pool in (s["keys"], s["values"]):
        pool[:, to] = torch.where(slot[:, None, :, None], pool[:, source], pool[:, to])
    if "bounds" in s:
        s["bounds"][:, to] = s["bounds"][:, source]


def _fork(s):
    ps, width = s["case"]["page"], s["width"]
    refs = s["refs"]
    refs.copy_(s["left"])
    parents = s["parents"].long()
    child = torch.arange(s["kept"], device="cuda")
    none = torch.full((s["batch"],), s["kept"], device="cuda")
    first = none.scatter_reduce(0, parents, child, "amin")[parents] == child
    n, held = s["lengths"].long()[parents], s["held"].long()[parents]
    full, need = n // ps, (n + 1 + ps - 1) // ps
    at = torch.arange(width, device="cuda")
    source = s["table"].long()[parents]
    share = at < full[:, None]
    alone = refs[source.clamp(min=0)] == 1
    stay = ~share & first[:, None] & (at < torch.minimum(held, need)[:, None]) & alone
    fresh = (at < need[:, None]) & ~share & ~stay
    order = (refs != 0).to(torch.int8).sort(stable=True)[1]  # free pages first
    free = (refs == 0).sum()
    rank = (fresh.flatten().cumsum(0) - 1).reshape(fresh.shape)
    page = torch.where(rank < free, order[rank.clamp(0, s["pages"] - 1)], -1)
    page = torch.where(fresh, page, source)
    taken = at < need[:, None]
    s["new_table"].copy_(torch.where(taken, page, s["new_table"].long()))
    s["new_lengths"].copy_(n)
    s["new_held"].copy_(need)
    gone = s["table"].long()[at < s["held"][:, None]]
    refs.index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    new = page[taken & (page >= 0)]
    refs.index_add_(0, new, torch.ones_like(new, dtype=torch.int32))
    cut = full.clamp(max=width - 1)[:, None]
    source, page, fresh = (x.gather(1, cut)[:, 0] for x in (source, page, fresh))
    parted = fresh & (n % ps != 0) & (page >= 0)
    listing = torch.stack((source, page, n % ps), -1)
    s["copies"].copy_(listing.masked_fill(~parted[:, None], -1))
    _copy(s, source[parted], page[parted], (n % ps)[parted])
    return _state(s)


def _compact(s):
    refs, limit, pages = s["refs"], s["case"]["limit"], s["pages"]
    refs.copy_(s["left"])
    s["table"].copy_(s["left_table"])
    at = torch.arange(pages, device="cuda")
    inside = torch.arange(s["width"], device="cuda") < s["held"][:, None]
    names = s["table"].long()[inside]
    count = torch.zeros_like(refs).index_add_(0, names, torch.ones_like(names, dtype=torch.int32))
    high = (at >= limit) & (refs > 0) & (refs == count)
    low = (at < limit) & (refs == 0)
    n = torch.minimum(high.sum(), low.sum()).clamp(max=s["copies"].shape[0])
    span = at[:s["copies"].shape[0]]
    source = (~high).to(torch.int8).sort(stable=True)[1][:span.shape[0]]
    to = (~low).to(torch.int8).sort(stable=True)[1][:span.shape[0]]
    live = span < n
    s["copies"].copy_(torch.stack((source, to, torch.full_like(to, s["case"]["page"])), -1)
                      .masked_fill(~live[:, None], -1))
    source, to = source[live], to[live]
    where = at.clone()
    where[source] = to
    s["table"].copy_(torch.where(inside, where[s["table"].long().clamp(min=0)],
                                 s["table"].long()))
    refs[to] = refs[source]
    refs[source] = 0
    _copy(s, source, to, torch.full_like(to, s["case"]["page"]))
    return _state(s)


def _beam(s):
    case = s["case"]
    batch, beams, keep, vocab = (case[k] for k in ("batch", "beams", "keep", "vocab"))
    x = s["logits"].float()
    value, token = x.sort(dim=-1, descending=True, stable=True)
    value, token = value[:, :keep].double(), token[:, :keep]
    top = value[:, :1]
    lse = top + torch.exp(x.double() - top).sum(-1, keepdim=True).log()
    score, length = s["scores"].double().reshape(-1, 1), s["lengths"].long().reshape(-1, 1)
    over = s["ended"].bool().reshape(-1, 1)
    rank = torch.arange(keep, device="cuda")
    total = torch.where(over, score.masked_fill(rank > 0, -math.inf), score + (value - lse))
    token = torch.where(over, EOS, token)
    grown = torch.where(over, length, length + 1)
    by = total / grown.clamp(min=1).double() ** case["power"]
    # candidates by (beam, token): ties go to the lowest
    place = torch.arange(batch * beams, device="cuda")[:, None] % beams * vocab + token
    flat = lambda v: v.expand(-1, keep).reshape(batch, -1)  # noqa: E731
    order = flat(place).sort(dim=-1, stable=True)[1]
    best = flat(by).gather(1, order).sort(dim=-1, descending=True, stable=True)[1]
    best = order.gather(1, best)[:, :keep]
    pad = keep - best.shape[1]
    total, grown, token, over = (flat(v).gather(1, best) for v in (total, grown, token, over))
    parent = best // keep + torch.arange(batch, device="cuda")[:, None] * beams
    live = total > -math.inf
    parent, token = parent.masked_fill(~live, -1), token.masked_fill(~live, -1)
    over = (over | (token == EOS)) & live
    grown = grown.masked_fill(~live, 0)
    assert pad <= 0
    for name, v in (("parents", parent), ("tokens", token), ("new_scores", total),
                    ("new_lengths", grown), ("new_ended", over)):
        s[name].copy_(v)
    flat = s["parents"].long().reshape(-1, 1)
    s["new_text"].copy_(torch.where(flat >= 0, s["text"][flat[:, 0].clamp(min=0)],
                                    s["new_text"]))
    return _state(s)


def run(state):
    if own:
        return _own(state)
    return {"tree": _attend, "verify": _verify, "fork": _fork, "compact": _compact,
            "beam": _beam}[state["kind"]](state)


# ---------------------------------------------------------- what it costs --

def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "beam":
        rows, kept = case["batch"] * (case["beams"] - case["ended"]), case["batch"] * case["keep"]
        if case["first"]:
            rows = case["batch"]
        return dict(bytes=rows * case["vocab"] * size + case["batch"] * case["beams"] * 12 +
                    kept * (20 + 8 * case["text"]), flops=3 * rows * case["vocab"])
    heads, kv, dim, layers = SHAPES[case["shape"]]
    per_row, ps = 2 * kv * dim * size, case["page"]
    if case["kind"] == "compact":
        moved = min((case["pages"] - case["limit"]) / 2, case["limit"] / 2)
        return dict(bytes=layers * moved * ps * 2 * per_row + case["pages"] * 6, flops=0)
    lengths = _lengths(case)
    if case["kind"] == "fork":
        parents, copied, entries = _parents(case), 0, 0
        for i, p in enumerate(parents):
            n = lengths[p // case["beams"]]
            entries += -(-(n + 1) // ps)
            copied += n % ps if p in parents[:i] else 0
        return dict(bytes=layers * copied * 2 * per_row + entries * 8 + len(parents) * 20, flops=0)
    counts = _counts(case)
    words = -(-case["nodes"] // 32)
    if case["kind"] == "verify":  # about one row behind the root moves in every sequence
        return dict(bytes=sum(counts) * (16 + 4 * words) + case["batch"] * 16 +
                    sum(c > 1 for c in counts) * layers * 2 * per_row, flops=0)
    rows = sum(n + m for n, m in zip(lengths, counts))
    pages = sum(-(-(n + m) // ps) for n, m in zip(lengths, counts))
    return dict(bytes=rows * per_row + sum(counts) * (heads * (2 * dim + 1) + words) * 4 +
                4 * pages, flops=4 * heads * dim * sum(m * (n + 1)
                                                       for n, m in zip(lengths, counts)))


# ------------------------------------------------- the definition, 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "verify": _exact_verify, "fork": _exact_fork,
            "compact": _exact_compact, "beam": _exact_beam}[case["kind"]](s, case)


def _line(parents, i):
    """Node i and its ancestors, in ascending order."""
    got = []
    while i >= 0:
        got.append(i)
        i = parents[i]
    return got[::-1]


def _exact_tree(s, case):
    heads, kv, dim, _ = SHAPES[case["shape"]]
    group, ps = heads // kv, case["page"]
    out = torch.zeros(s["total"], heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((s["total"], heads), -math.inf, dtype=torch.float64, device="cuda")
    begin = 0
    for b, (n, m) in enumerate(zip(_lengths(case), _counts(case))):
        if m == 0:
            continue
        parents = s["parents"][begin:begin + m].tolist()
        hide = torch.full((m, n + m), -math.inf, dtype=torch.float64)
        hide[:, :n] = 0.0
        for i in range(m):
            hide[i, [n + j for j in _line(parents, i)]] = 0.0
        hide = hide.cuda()
        row = torch.arange(n + m, device="cuda")
        page, slot = s["table"][b].long()[row // ps], row % ps
        for h in range(kv):
            k, v = s["keys"][0][page, h, slot].double(), s["values"][0][page, h, slot].double()
            for g in range(h * group, (h + 1) * group):
                score = s["query"][begin:begin + m, g].double() @ k.T.contiguous() * s["scale"]
                score += hide
                total = torch.logsumexp(score, -1)
                lse[begin:begin + m, g] = total
                out[begin:begin + m, g] = torch.exp(score - total[:, None]) @ v
        begin += m
    return dict(out=out, lse=lse)


def _exact_verify(s, case):
    ps, begin = case["page"], 0
    keys, values, bounds = s["keys"].double(), s["values"].double(), s["bounds"].double()
    for b, (n, m) in enumerate(zip(_lengths(case), _counts(case))):
        parents, tokens, chosen = (s[k][begin:begin + m].tolist()
                                   for k in ("parents", "tokens", "chosen"))
        begin += m
        path = [0] if m else []
        while path:
            after = [j for j in range(m) if parents[j] == path[-1] and
                     tokens[j] == chosen[path[-1]]]
            if not after:
                break
            path.append(after[0])
        table = s["table"][b].tolist()
        for k, i in enumerate(path):
            if i == k:
                continue
            source, to = table[(n + i) // ps], table[(n + k) // ps]
            for pool in (keys, values):
                pool[:, to, :, (n + k) % ps] = pool[:, source, :, (n + i) % ps]
            row = keys[:, to, :, (n + k) % ps]
            bounds[:, to, :, 0] = torch.minimum(bounds[:, to, :, 0], row)
            bounds[:, to, :, 1] = torch.maximum(bounds[:, to, :, 1], row)
    return dict(mask=None, depths=None, path=None, counts=None, last=None, new_lengths=None,
                keys=keys, values=values, bounds=bounds)


def _exact_fork(s, case):
    ps = case["page"]
    keys, values, bounds = s["keys"].double(), s["values"].double(), s["bounds"].double()
    refs, table, lengths = s["left"].tolist(), s["table"].tolist(), s["lengths"].tolist()
    held, free, seen = s["held"].tolist(), [p for p, r in enumerate(refs) if r == 0], set()
    for p in s["parents"].tolist():
        n = lengths[p]
        for c in range(n // ps, -(-(n + 1) // ps)):
            mine = p not in seen and c < held[p] and refs[table[p][c]] == 1
            page = table[p][c] if mine else free.pop(0)
            if not mine and c == n // ps and n % ps:
                for pool in (keys, values):
                    pool[:, page, :, :n % ps] = pool[:, table[p][c], :, :n % ps]
                bounds[:, page] = bounds[:, table[p][c]]
        seen.add(p)
    return dict(refs=None, new_table=None, new_lengths=None, new_held=None, copies=None,
                keys=keys, values=values, bounds=bounds)


def _exact_compact(s, case):
    keys, values = s["keys"].double(), s["values"].double()
    refs, limit = s["left"].tolist(), case["limit"]
    high = [p for p in range(limit, len(refs)) if refs[p]]
    low = [p for p in range(limit) if not refs[p]]
    for source, to in zip(high, low):
        keys[:, to], values[:, to] = keys[:, source], values[:, source]
    return dict(refs=None, table=None, copies=None, keys=keys, values=values)


def _exact_beam(s, case):
    beams, keep = case["beams"], case["keep"]
    got = torch.full((case["batch"], keep), -math.inf, dtype=torch.float64, device="cuda")
    for r in range(case["batch"]):
        x = s["logits"][r * beams:(r + 1) * beams].double()
        score = s["scores"][r].double()[:, None]
        length = s["lengths"][r].double()[:, None].expand(-1, x.shape[1]) + 1
        total = score + torch.log_softmax(x, -1)
        for i in range(beams):
            if s["ended"][r, i]:
                total[i] = -math.inf
                total[i, EOS] = score[i, 0]
                length = length.clone()
                length[i] -= 1
        by = (total / length.clamp(min=1) ** case["power"]).flatten()
        best = by.topk(keep)[1]
        got[r] = total.flatten()[best]
    return dict(parents=None, tokens=None, new_scores=got, new_lengths=None, new_ended=None,
                new_text=None)
