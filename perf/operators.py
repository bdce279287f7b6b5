"""Performance cases of the paged KV cache: append, attention of one new token,
page selection with sparse attention, and eviction by accumulated weight.

``run`` computes a case with elementary torch operations in 32 bits (64 where
whole numbers hang on them), or, with ``own``, through the framework's entry
points. The shapes are the repository's synthetic workloads (the TinyLlama
and Llama-2-7B attention shapes, the small test shapes) and a generic odd one.

Inputs come from the seed alone. Keys drift slowly along a sequence, so that
some pages matter more to a query than others; rows behind a sequence's end
hold what an earlier sequence left there; pages lie in no order.
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

SHAPES = {
    "tiny": (4, 2, 16),
    "step_gqa2": (4, 2, 64),
    "step_gqa4": (8, 2, 64),
    "step_mha128": (2, 2, 128),
    "tinyllama": (32, 4, 64),
    "llama7b": (32, 32, 128),
    "odd": (24, 3, 80),  # a generic width that no power of two divides into
}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MOST_BYTES = 2.2e9  # of one case's cached rows


def listed():
    return [
        # one chat, a short context: the smallest call, where latency counts
        dict(name="attend_chat", kind="attend", shape="tinyllama", type="f32", batch=1, low=37,
             high=37, page=16, order="head", idle=0),
        # an ordinary serving batch: lengths from one token to 2,048, two idle slots
        dict(name="attend_batch", kind="attend", shape="tinyllama", type="bf16", batch=32, low=1,
             high=2048, page=16, order="head", idle=2),
        # long documents on the 7B widths, one KV head per query head
        dict(name="attend_long", kind="attend", shape="llama7b", type="f16", batch=4, low=24000,
             high=32768, page=64, order="head", idle=0),
        # odd sizes: 80 dims, pages of 24 rows, the heads of a row side by side
        dict(name="attend_odd", kind="attend", shape="odd", type="f32", batch=7, low=300,
             high=5001, page=24, order="slot", idle=0),
        # a batch whose attention weights are added up for a later eviction
        dict(name="weigh_batch", kind="weigh", shape="tinyllama", type="bf16", batch=16, low=500,
             high=4096, page=32, order="head", idle=0),
        # one long chat that reads the pages that matter
        dict(name="sparse_chat", kind="sparse", shape="step_gqa4", type="f32", batch=1, low=8001,
             high=8001, page=16, order="head", idle=0, top=32, first=1, last=2),
        # a batch of long contexts, a sixteenth of each read
        dict(name="sparse_long", kind="sparse", shape="tinyllama", type="bf16", batch=16,
             low=16000, high=32768, page=32, order="head", idle=0, top=64, first=1, last=2),
        # a decode step's eviction: a few rows over the budget
        dict(name="evict_step", kind="evict", shape="tinyllama", type="bf16", batch=16, low=1025,
             high=1040, page=16, order="head", idle=0, budget=1024, first=4, last=128,
             shuffled=True),
        # long prompts cut down to a budget after they were read
        dict(name="evict_prompt", kind="evict", shape="llama7b", type="f16", batch=4, low=6000,
             high=8192, page=64, order="head", idle=0, budget=2048, first=4, last=256,
             shuffled=False),
        # one new token for each sequence of a full batch
        dict(name="append_tokens", kind="append", shape="tinyllama", type="bf16", batch=64, low=0,
             high=2000, page=16, order="head", idle=0, new=1),
        # several prompts at once, ragged, behind what their sequences hold
        dict(name="append_prompts", kind="append", shape="llama7b", type="f16", batch=8, low=0,
             high=500, page=64, order="head", idle=0, new=2048),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "weigh", "sparse", "sparse", "evict", "evict",
                       "append"])
    shape = rng.choice(["tiny", "step_gqa2", "step_gqa4", "step_mha128", "tinyllama", "tinyllama",
                        "llama7b", "llama7b", "odd"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    case = dict(kind=kind, shape=shape, type=dtype, batch=_log_int(rng, 1, 64),
                page=rng.choice([8, 16, 16, 24, 32, 64, 128]),
                order=rng.choice(["head", "head", "slot"]))
    case["idle"] = rng.choice([0, 0, case["batch"] // 8])
    heads, kv, dim = SHAPES[shape]
    row = 2 * kv * dim * (4 if dtype == "f32" else 2)
    most = int(MOST_BYTES / 2 / row / case["batch"])
    if kind == "append":
        case["high"] = _log_int(rng, 1, min(2000, max(2, most)))
        case["low"] = rng.randint(0, case["high"])
        case["new"] = 1 if rng.random() < 0.5 else _log_int(rng, 2, max(2, min(2000, most // 4)))
        return case
    if kind == "evict":
        case["high"] = _log_int(rng, 64, min(8000, max(65, most // 2)))
        case["low"] = rng.randint(case["high"] // 2, case["high"])
        case["budget"] = rng.choice([max(16, case["high"] - rng.randint(1, 40)),
                                     _log_int(rng, 16, case["high"])])
        case["first"] = rng.randint(0, 4)
        case["last"] = rng.randint(1, max(1, case["budget"] // 4))
        case["shuffled"] = rng.random() < 0.5
        return case
    case["high"] = _log_int(rng, 1, min(32768, most))
    case["low"] = rng.randint(1, case["high"])
    if kind == "weigh":
        case["high"] = min(case["high"], 16384)
        case["low"] = min(case["low"], case["high"])
    if kind == "sparse":
        case["top"] = _log_int(rng, 4, 128)
        case["first"], case["last"] = rng.randint(0, 1), rng.randint(1, 3)
    return case


# ------------------------------------------------------------------ inputs --

def _lengths(case):
    """Rows of each sequence: spread evenly over the case's range, idle ones at the end."""
    n, low, high = case["batch"] - case["idle"], case["low"], case["high"]
    spread = [high if i == 0 else low + int((i * 0.6180339887) % 1.0 * (high - low + 1))
              for i in range(n)]
    return spread + [0] * case["idle"]


def _new_rows(case):
    """Rows that each sequence gains in an append."""
    if case["new"] == 1:
        return [1] * case["batch"]
    return [case["new"] if i == 0 else int((i * 0.7548776662) % 1.0 * case["new"]) + 1
            if i < case["batch"] - case["idle"] else 0 for i in range(case["batch"])]


def _gen(seed, stream):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + stream)


def _normal(seed, stream, *shape, sigma=1.0):
    return torch.randn(*shape, generator=_gen(seed, stream), device="cuda") * sigma


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pool(case, pages, seed, stream):
    """Rows of every page, [pages, kv_heads, page, dim] whichever way they lie, with a drift
    that a page's rows share."""
    heads, kv, dim = SHAPES[case["shape"]]
    ps, dtype = case["page"], DTYPES[case["type"]]
    rows = torch.empty(pages, kv, ps, dim, device="cuda", dtype=dtype)
    rows.normal_(0.0, 0.9, generator=_gen(seed, stream))
    rows += _normal(seed, stream + 1, pages, kv, 1, dim, sigma=0.5).to(dtype)
    if case["order"] == "slot":
        return rows.transpose(1, 2).contiguous().transpose(1, 2)
    return rows


def prepare(case, seed):
    heads, kv, dim = SHAPES[case["shape"]]
    ps, batch, kind = case["page"], case["batch"], case["kind"]
    lengths = _lengths(case)
    new = _new_rows(case) if kind == "append" else [0] * batch
    longest = max(n + m for n, m in zip(lengths, new))
    width = -(-longest // ps)  # pages of each sequence's table
    pages = batch * width + 3
    order = torch.randperm(pages, generator=_gen(seed, 1), device="cuda")
    s = dict(kind=kind, case=case, page=ps, batch=batch, heads=heads, kv=kv, dim=dim, width=width,
             pages=pages, longest=longest, scale=dim ** -0.5, lengths=_ints(lengths),
             table=order[:batch * width].reshape(batch, width).int().contiguous(),
             keys=_pool(case, pages, seed, 10), values=_pool(case, pages, seed, 20))
    if kind != "append":
        s["query"] = _normal(seed, 30, batch, heads, dim, sigma=1.5)
        s["out"] = torch.empty(batch, heads, dim, device="cuda")
        s["lse"] = torch.empty(batch, heads, device="cuda")
    if kind in ("sparse", "append"):
        s["bounds"] = torch.stack((s["keys"].amin(2), s["keys"].amax(2)), 2)
    if kind == "sparse":
        s["selected"] = torch.empty(batch, kv, case["top"], dtype=torch.int32, device="cuda")
    if kind in ("weigh", "evict", "append"):
        # weights and positions of the rows: a few rows hold most of the weight, new ones none
        s["stride"] = longest
        w = _normal(seed, 40, batch, kv, longest, sigma=2.0).exp_()
        w *= torch.rand(batch, kv, longest, generator=_gen(seed, 41), device="cuda") > 0.05
        at = torch.arange(longest, device="cuda").expand(batch, kv, longest)
        if case.get("shuffled"):  # rows that earlier evictions moved, with gaps between them
            at = torch.rand(batch, kv, longest, generator=_gen(seed, 42), device="cuda")
            inside = torch.arange(longest, device="cuda") < s["lengths"][:, None, None]
            at = at.masked_fill(~inside, 2.0).argsort(-1).argsort(-1) * 3 + 1
        s["left"] = torch.stack((w.view(torch.int32), at.int()))
        s["history"] = s["left"].clone()
        s["weights"], s["positions"] = s["history"][0].view(torch.float32), s["history"][1]
    if kind in ("evict", "append"):
        s["new_lengths"] = torch.empty_like(s["lengths"])
    if kind == "append":
        starts = [sum(new[:i]) for i in range(batch + 1)]
        s["most"], s["ragged"] = max(new), case["new"] > 1
        s["starts"], s["firsts"] = _ints(starts), _ints([n + 100 for n in lengths])
        s["new_keys"] = _normal(seed, 50, starts[-1], kv, dim)
        s["new_values"] = _normal(seed, 51, starts[-1], kv, dim)
    if own:
        _handles(s)
    return s


# ------------------------------------------------- the framework's kernels --

class _Buffer:
    """A torch tensor as the device buffer that the entry points take."""

    def __init__(self, tensor):
        self.tensor = tensor
        self.nbytes = tensor.numel() * tensor.element_size()
        self.ptr = ctypes.c_void_p(tensor.data_ptr())


def _handles(s):
    """The views of the cache and its sequences, and the workspace, that a program keeps."""
    import nutllm_amd as nut

    case = s["case"]
    b = {k: _Buffer(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
    s["b"] = b
    s["paged"] = nut.PagedKV(
        b["keys"], b["values"], s["pages"], case["page"], s["kv"], s["dim"],
        {"f32": nut.F32, "f16": nut.F16, "bf16": nut.BF16}[case["type"]],
        strides=s["keys"].stride()[:3], bounds=b.get("bounds"))
    s["seqs"] = nut.PagedBatch(b["table"], s["width"], b["lengths"], s["batch"], s["longest"])
    if "weights" in b:
        s["kept"] = nut.PagedHistory(b["weights"], b["positions"], s["stride"])
    need = {"attend": lambda: s["paged"].attention_workspace(s["seqs"], s["heads"]),
            "weigh": lambda: s["paged"].attention_workspace(s["seqs"], s["heads"], weighted=True),
            "sparse": lambda: max(s["paged"].select_workspace(s["seqs"], s["heads"], case["top"]),
                                  s["paged"].attention_workspace(s["seqs"], s["heads"],
                                                                 top=case["top"])),
            "evict": lambda: s["paged"].evict_workspace(s["seqs"], case["budget"]),
            "append": lambda: 0}[s["kind"]]()
    s["space"] = _Buffer(torch.empty(max(1, need), dtype=torch.uint8, device="cuda"))


def _own(s):
    case, b, kind, paged = s["case"], s["b"], s["kind"], s["paged"]
    if kind == "append":
        paged.append(s["seqs"], b["new_keys"], b["new_values"], b["new_lengths"],
                     starts=b["starts"] if s["ragged"] else None, max_new=s["most"],
                     history=s["kept"], first_positions=b["firsts"])
        return _state(s)
    if kind == "evict":
        s["history"].copy_(s["left"])  # what attention left since the last eviction
        paged.evict(s["seqs"], s["kept"], b["new_lengths"], case["budget"], first=case["first"],
                    last=case["last"], workspace=s["space"])
        return _state(s)
    if kind == "sparse":
        paged.select(s["seqs"], b["query"], b["selected"], s["heads"], case["top"],
                     first=case["first"], last=case["last"], workspace=s["space"])
        paged.attention(s["seqs"], b["query"], b["out"], s["heads"], scale=s["scale"],
                        lse=b["lse"], selected=b["selected"], top=case["top"],
                        workspace=s["space"])
        return dict(out=s["out"], lse=s["lse"], selected=s["selected"])
    paged.attention(s["seqs"], b["query"], b["out"], s["heads"], scale=s["scale"], lse=b["lse"],
                    history=s["kept"] if kind == "weigh" else None, workspace=s["space"])
    got = dict(out=s["out"], lse=s["lse"])
    return dict(got, weights=s["weights"]) if kind == "weigh" else got


# ------------------------------------------------------------- plain forms --

def _state(s):
    got = {k: s[k] for k in ("keys", "values", "weights", "positions", "new_lengths")}
    return dict(got, bounds=s["bounds"]) if "bounds" in s else got


def _rows(pool, table):
    """[batch, kv, rows, dim] of the pages that a table names, in 32 bits."""
    b, w = table.shape
    got = pool[table.long()].transpose(1, 2)  # [b, kv, w, page, dim]
    return got.reshape(b, got.shape[1], -1, got.shape[-1]).float()


def _softmax(query, k, v, seen, scale, kv):
    """out, lse and the weights of a query's heads over rows [batch, kv, rows, dim]."""
    b, heads, dim = query.shape
    q = query.reshape(b, kv, heads // kv, dim) * scale
    score = torch.matmul(q, k.transpose(-1, -2)).masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
    z = p.sum(-1, keepdim=True)
    safe = z.masked_fill(z == 0.0, 1.0)
    out = torch.matmul(p, v.masked_fill(~seen.transpose(-1, -2), 0.0)) / safe
    return out.reshape(b, heads, dim), (top + z.log()).reshape(b, heads), p / safe


def _attend(s):
    rows = s["width"] * s["page"]
    seen = torch.arange(rows, device="cuda") < s["lengths"][:, None, None, None]
    out, lse, p = _softmax(s["query"], _rows(s["keys"], s["table"]),
                           _rows(s["values"], s["table"]), seen, s["scale"], s["kv"])
    if s["kind"] != "weigh":
        return dict(out=out, lse=lse)
    s["weights"] += p.sum(2)[..., :s["longest"]]
    return dict(out=out, lse=lse, weights=s["weights"])


def _sparse(s):
    case, b, kv, ps = s["case"], s["batch"], s["kv"], s["page"]
    top = case["top"]
    q = s["query"].reshape(b, kv, -1, s["dim"]).double()
    bounds = s["bounds"][s["table"].long()].transpose(1, 2).double()  # [b, kv, w, 2, dim]
    lo, hi = bounds[..., 0, :], bounds[..., 1, :]
    score = (torch.matmul(q.clamp(min=0), hi.transpose(-1, -2)) +
             torch.matmul(q.clamp(max=0), lo.transpose(-1, -2))).amax(2)
    count = ((s["lengths"] + ps - 1) // ps)[:, None, None]
    at = torch.arange(s["width"], device="cuda")
    score = score.masked_fill((at < case["first"]) | (at >= count - case["last"]), math.inf)
    score = score.masked_fill(at >= count, -math.inf)
    best = score.sort(dim=-1, descending=True, stable=True)[1][..., :top]
    best = best.masked_fill(best >= count, s["width"]).sort(-1)[0]
    best = torch.nn.functional.pad(best, (0, top - best.shape[-1]), value=s["width"])
    none = best == s["width"]
    selected = best.masked_fill(none, -1).int()
    at = best.masked_fill(none, 0)
    page = s["table"].long().gather(1, at.reshape(b, -1)).reshape(b, kv, top)
    head = torch.arange(kv, device="cuda")[None, :, None]
    k = s["keys"][page, head].reshape(b, kv, top * ps, s["dim"]).float()
    v = s["values"][page, head].reshape(b, kv, top * ps, s["dim"]).float()
    row = at[..., None] * ps + torch.arange(ps, device="cuda")
    seen = (row < s["lengths"][:, None, None, None]) & ~none[..., None]
    out, lse, _ = _softmax(s["query"], k, v, seen.reshape(b, kv, 1, -1), s["scale"], kv)
    return dict(out=out, lse=lse, selected=selected)


def _evict(s):
    case, b, kv, ps = s["case"], s["batch"], s["kv"], s["page"]
    budget = min(case["budget"], s["longest"])
    s["history"].copy_(s["left"])
    n = s["lengths"][:, None, None]
    at = torch.arange(s["longest"], device="cuda")
    inside = at < n
    pos = s["positions"]
    newest = pos.masked_fill(~inside, -1).amax(-1, keepdim=True)
    key = s["weights"].masked_fill((pos < case["first"]) | (pos > newest - case["last"]), math.inf)
    key = key.masked_fill(~inside, -math.inf)
    best = key.sort(dim=-1, descending=True, stable=True)[1][..., :budget]
    kept = torch.zeros_like(inside.expand(b, kv, -1)).scatter(-1, best, True) & inside
    over = kept & (at >= budget)
    order = (~over).to(torch.int8).sort(dim=-1, stable=True)[1]  # rows beyond the budget first
    hole = ~kept[..., :budget] & inside[..., :budget]
    rank = (hole.cumsum(-1) - 1).clamp(min=0)
    to = at[:budget].expand(b, kv, budget)
    source = torch.where(hole, order.gather(-1, rank), to)
    head = torch.arange(kv, device="cuda")[None, :, None]
    table = s["table"].long()
    seq = torch.arange(b, device="cuda")[:, None, None]
    from_page, to_page = table[seq, source // ps], table[seq, to // ps]
    for pool in (s["keys"], s["values"]):
        pool[to_page, head, to % ps] = pool[from_page, head, source % ps]
    s["history"][..., :budget] = s["history"].gather(-1, source.expand(2, b, kv, budget))
    torch.clamp(s["lengths"], max=case["budget"], out=s["new_lengths"])
    return _state(s)


def _append(s):
    ps, dtype = s["page"], s["keys"].dtype
    row = torch.arange(s["new_keys"].shape[0], device="cuda")
    starts, lengths = s["starts"].long(), s["lengths"].long()
    seq = torch.searchsorted(starts[1:], row, right=True)
    j = row - starts[seq]
    at = lengths[seq] + j
    page = s["table"].long()[seq, at // ps]
    k, v = s["new_keys"].to(dtype), s["new_values"].to(dtype)
    s["keys"][page, :, at % ps] = k
    s["values"][page, :, at % ps] = v
    fresh = (at // ps * ps >= lengths[seq])[:, None, None]
    lo, hi = (x.contiguous() for x in s["bounds"].float().unbind(2))
    lo[page] = torch.where(fresh, math.inf, lo[page])
    hi[page] = torch.where(fresh, -math.inf, hi[page])
    lo.index_reduce_(0, page, k.float(), "amin")
    hi.index_reduce_(0, page, k.float(), "amax")
    s["bounds"].copy_(torch.stack((lo, hi), 2))
    s["weights"][seq, :, at] = 0.0
    s["positions"][seq, :, at] = (s["firsts"].long()[seq] + j).int()[:, None]
    torch.add(s["lengths"], s["starts"].diff(), out=s["new_lengths"])
    return _state(s)


def run(state):
    if own:
        return _own(state)
    return {"attend": _attend, "weigh": _attend, "sparse": _sparse, "evict": _evict,
            "append": _append}[state["kind"]](state)


# ---------------------------------------------------------- what it costs --

def work(case):
    heads, kv, dim = SHAPES[case["shape"]]
    size, ps, lengths = 4 if case["type"] == "f32" else 2, case["page"], _lengths(case)
    rows, pages = sum(lengths), sum(-(-n // ps) for n in lengths)
    per_row = 2 * kv * dim * size
    ends = case["batch"] * heads * (2 * dim + 1) * 4 + 4 * pages
    if case["kind"] == "append":
        new = _new_rows(case)
        touched = sum((n + m - 1) // ps - n // ps + 1 for n, m in zip(lengths, new) if m)
        return dict(bytes=sum(new) * (per_row + 8 * kv * dim + 8 * kv) +
                    touched * per_row + 8 * case["batch"], flops=0)
    if case["kind"] == "evict":
        budget, kept = case["budget"], case["first"] + case["last"]
        moved = sum(min(case["last"], n - budget) + max(0, budget - kept) *
                    max(0, n - budget - case["last"]) / max(1, n - kept)
                    for n in lengths if n > budget)
        return dict(bytes=rows * kv * 8 + moved * (2 * per_row + 16 * kv), flops=0)
    if case["kind"] == "sparse":
        read = sum(min(n, case["top"] * ps) for n in lengths)
        return dict(bytes=read * per_row + pages * per_row + ends,
                    flops=4 * heads * dim * (read + pages))
    more = 8 * rows * kv if case["kind"] == "weigh" else 0
    return dict(bytes=rows * per_row + ends + more, flops=4 * rows * heads * dim)


# ------------------------------------------------- the definition, 64 bits --

def _one(q, k, v, scale):
    """out, lse and weights of heads [g, dim] over rows [n, dim], all in 64 bits."""
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.full_like(q[:, 0], -math.inf), q.new_zeros(len(q), 0)
    score = (k @ q.T).T * scale
    lse = torch.logsumexp(score, -1)
    p = torch.exp(score - lse[:, None])
    return (v.T @ p.T).T, lse, p


def exact(case, seed):
    s = prepare(case, seed)
    heads, kv, dim = SHAPES[case["shape"]]
    ps, group, kind = case["page"], heads // kv, case["kind"]
    lengths, table = _lengths(case), s["table"].tolist()
    if kind == "append":
        return _exact_append(s, case, lengths)
    if kind == "evict":
        return _exact_evict(s, case, lengths)
    out = torch.zeros(case["batch"], heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((case["batch"], heads), -math.inf, dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if kind == "weigh" else None
    for b, n in enumerate(lengths):
        ids = torch.tensor(table[b][:-(-n // ps)], dtype=torch.long, device="cuda")
        for h in range(kv):
            mine = slice(h * group, (h + 1) * group)
            q = s["query"][b, mine].double()
            use, here = ids, torch.arange(len(ids), device="cuda")
            if kind == "sparse" and len(ids) > case["top"]:
                bound = s["bounds"][ids, h].double()  # [pages, 2, dim]
                score = torch.maximum(q[:, None] * bound[None, :, 0],
                                      q[:, None] * bound[None, :, 1]).sum(-1).amax(0)
                score[:case["first"]] = math.inf
                score[len(ids) - case["last"]:] = math.inf
                here = score.argsort(descending=True, stable=True)[:case["top"]].sort()[0]
                use = ids[here]
            keep = (here[:, None] * ps + torch.arange(ps, device="cuda")).reshape(-1) < n
            k = s["keys"][use, h].reshape(-1, dim)[keep].double()
            v = s["values"][use, h].reshape(-1, dim)[keep].double()
            out[b, mine], lse[b, mine], p = _one(q, k, v, s["scale"])
            if weights is not None:
                weights[b, h, :n] += p.sum(0)
    got = dict(out=out, lse=lse)
    if kind == "sparse":
        return dict(got, selected=None)
    return dict(got, weights=weights) if weights is not None else got


def _exact_append(s, case, lengths):
    ps, new, row = case["page"], _new_rows(case), 0
    keys, values, bounds = s["keys"].double(), s["values"].double(), s["bounds"].double()
    weights = s["weights"].double()
    for b, (n, m) in enumerate(zip(lengths, new)):
        for c in range(n // ps, (n + m - 1) // ps + 1 if m else 0):
            page, begin, end = int(s["table"][b, c]), max(n, c * ps), min(n + m, (c + 1) * ps)
            k = s["new_keys"][row + begin - n:row + end - n].double().transpose(0, 1)
            slots = slice(begin - c * ps, end - c * ps)
            keys[page, :, slots] = k
            values[page, :, slots] = \
                s["new_values"][row + begin - n:row + end - n].double().transpose(0, 1)
            lo, hi = k.amin(1), k.amax(1)
            if n > c * ps:
                lo, hi = torch.minimum(lo, bounds[page, :, 0]), torch.maximum(hi, bounds[page, :, 1])
            bounds[page, :, 0], bounds[page, :, 1] = lo, hi
        weights[b, :, n:n + m] = 0.0
        row += m
    return dict(keys=keys, values=values, bounds=bounds, weights=weights, positions=None,
                new_lengths=None)


def _exact_evict(s, case, lengths):
    ps, budget, table = case["page"], case["budget"], s["table"].tolist()
    keys, values, weights = s["keys"].double(), s["values"].double(), s["weights"].double()
    for b, n in enumerate(lengths):
        if n <= budget:
            continue
        pages = torch.tensor(table[b], device="cuda")
        for h, (w, pos) in enumerate(zip(s["weights"][b, :, :n].tolist(),
                                         s["positions"][b, :, :n].tolist())):
            newest = max(pos)
            free = [not (p < case["first"] or p > newest - case["last"]) for p in pos]
            rank = sorted(range(n), key=lambda i: (free[i], -w[i] if free[i] else 0.0, i))
            kept = set(rank[:budget])
            holes = torch.tensor([i for i in range(budget) if i not in kept], dtype=torch.long,
                                 device="cuda")
            moved = torch.tensor([i for i in range(budget, n) if i in kept], dtype=torch.long,
                                 device="cuda")
            for pool in (keys, values):
                pool[pages[holes // ps], h, holes % ps] = pool[pages[moved // ps], h, moved % ps]
            weights[b, h, holes] = weights[b, h, moved]
    return dict(keys=keys, values=values, weights=weights, positions=None, new_lengths=None)
