"""The decoder block's operators around its quantized projections, as they are
measured: appending rotated keys to a paged cache, attention of drafted
tokens over it, keeping the accepted ones, and the norms between blocks.

Each of B sequences holds lengths[b] tokens in pages that its row of the page
table names, and T drafted tokens (a tree, a chain, or a single one), of which
counts[b] are in use. Inputs are made on the GPU from the seed; lengths and
counts follow from the case, so that its work does.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "bf16": 2}
_EPSILON = 1e-5
_THETA = 500000.0
_NO_PAGE = 0xFFFFFFFF


def listed():
    return [
        # One token of one conversation through a Llama-8B-shaped block: the
        # smallest call, where latency counts.
        {"name": "attention_one_token", "kind": "attention", "B": 1, "T": 1, "heads": 32, "kv": 8, "dim": 128,
         "length": 777, "page": 16, "tree": False, "dtype": "bf16"},
        # A decode batch of 32 conversations of different lengths, no drafts.
        {"name": "attention_decode_b32", "kind": "attention", "B": 32, "T": 1, "heads": 32, "kv": 8, "dim": 128,
         "length": 4096, "page": 64, "tree": False, "dtype": "bf16"},
        # Trees of 24 drafted tokens of 8 conversations, small pages.
        {"name": "attention_tree_b8", "kind": "attention", "B": 8, "T": 24, "heads": 32, "kv": 8, "dim": 128,
         "length": 8192, "page": 16, "tree": True, "dtype": "bf16"},
        # The largest: trees of 64 over long contexts, a 70B-shaped block.
        {"name": "attention_tree_b16_long", "kind": "attention", "B": 16, "T": 64, "heads": 64, "kv": 8, "dim": 128,
         "length": 16384, "page": 64, "tree": True, "dtype": "bf16"},
        # Odd sizes in f32: 7 drafted tokens, five query heads to a key head,
        # narrow heads, pages of 48, and a conversation that only begins.
        {"name": "attention_odd_f32", "kind": "attention", "B": 3, "T": 7, "heads": 20, "kv": 4, "dim": 80,
         "length": 1501, "page": 48, "tree": True, "dtype": "f32"},
        # The append of one token: the f32 projections of one row.
        {"name": "append_one_token", "kind": "append", "B": 1, "T": 1, "heads": 32, "kv": 8, "dim": 128, "rotary": 128,
         "length": 777, "page": 16, "tree": False, "interleaved": False, "x": "f32", "dtype": "bf16"},
        # Trees of 64 of 16 conversations, a 70B-shaped block's projections.
        {"name": "append_tree_b16", "kind": "append", "B": 16, "T": 64, "heads": 64, "kv": 8, "dim": 128,
         "rotary": 128, "length": 1024, "page": 64, "tree": True, "interleaved": False, "x": "f32", "dtype": "bf16"},
        # Prompts of 1000 tokens; half of each narrow head rotated, in
        # neighbouring pairs, into an f32 cache.
        {"name": "append_prompt_f32", "kind": "append", "B": 4, "T": 1000, "heads": 20, "kv": 4, "dim": 80,
         "rotary": 40, "length": 300, "page": 48, "tree": False, "interleaved": True, "x": "bf16", "dtype": "f32"},
        # Keeping the accepted tokens: one conversation, one layer's cache.
        {"name": "commit_one", "kind": "commit", "layers": 1, "B": 1, "T": 24, "keep": 6, "kv": 8, "dim": 128,
         "length": 777, "page": 16, "dtype": "bf16"},
        # The same of 32 conversations in every layer of a 32-layer model.
        {"name": "commit_b32_layers", "kind": "commit", "layers": 32, "B": 32, "T": 24, "keep": 6, "kv": 8, "dim": 128,
         "length": 100, "page": 16, "dtype": "bf16"},
        # The norm before a block with the residual add of the one before it:
        # one token, bf16 stream, f32 projection, bf16 into the next one.
        {"name": "norm_one_token", "kind": "norm", "M": 1, "width": 4096, "stream": "bf16", "update": "f32",
         "out": "bf16", "post": False, "gate": None, "scale": 1.0},
        # Norms before and after a block with a gate per value, for a prompt
        # of 2048 tokens of a 70B-shaped model with an f32 stream.
        {"name": "norm_sandwich_prompt", "kind": "norm", "M": 2048, "width": 8192, "stream": "f32", "update": "f32",
         "out": "bf16", "post": True, "gate": "rows", "scale": 0.5},
    ]


def _log(rng, low, high, step=1):
    """A multiple of step from low to high, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / step)) * step))


def draw(rng: random.Random):
    kind = rng.choice(["attention"] * 5 + ["append"] * 3 + ["norm"] * 3 + ["commit"])
    if kind == "norm":
        case = {"kind": kind, "M": _log(rng, 1, 4096), "width": _log(rng, 256, 16384, rng.choice([1, 64, 64])),
                "stream": rng.choice(["bf16", "f32"]), "update": rng.choice(["f32", "f32", "bf16"]),
                "out": rng.choice(["bf16", "bf16", "f32"]), "post": rng.random() < 0.5,
                "gate": rng.choice([None, None, "columns", "rows"]), "scale": rng.choice([1.0, 0.5, 0.22])}
        while case["M"] * case["width"] > 2048 * 8192:
            case["M"] //= 2
        return case
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    case = {"kind": kind, "kv": rng.choice([1, 2, 4, 8, 8]), "dim": dim, "dtype": rng.choice(["bf16", "bf16", "f32"]),
            "page": rng.choice([16, 16, 32, 48, 64, 128, 256])}
    if kind == "commit":
        keep = rng.randint(1, 12)
        return case | {"layers": rng.choice([1, 2, 8, 16]), "B": _log(rng, 1, 32), "T": rng.randint(2 * keep, 3 * keep + 8),
                       "keep": keep, "length": _log(rng, 1, 100)}
    case["heads"] = case["kv"] * rng.choice([1, 2, 4, 4, 5, 8])
    if kind == "append":
        case |= {"B": _log(rng, 1, 32), "T": _log(rng, 1, 1024), "x": rng.choice(["f32", "f32", "bf16"]),
                 "rotary": rng.choice([dim, dim, dim // 2]), "length": _log(rng, 1, 1024),
                 "tree": rng.random() < 0.5, "interleaved": rng.random() < 0.3}
        while case["B"] * case["T"] * (case["heads"] + 2 * case["kv"]) * dim > 16 * 64 * 80 * 128:
            case["T"] = max(1, case["T"] // 2)
            case["B"] = max(1, case["B"] * 3 // 4)
        return case
    case |= {"B": _log(rng, 1, 64), "T": _log(rng, 1, 128), "length": _log(rng, 1, 16384), "tree": rng.random() < 0.7}
    # The largest listed case bounds it; f32 products run at a sixteenth of bf16's rate.
    top = work(next(c for c in listed() if c["name"] == "attention_tree_b16_long"))
    least = 1 if case["dtype"] == "bf16" else 16
    while work(case)["bytes"] > top["bytes"] or work(case)["flops"] * least > top["flops"]:
        case["length"] = max(1, case["length"] * 2 // 3)
        case["B"] = max(1, case["B"] * 3 // 4)
    return case


# ---- what follows from the case alone ----

def _lengths(case):
    """Committed tokens of each sequence: from a quarter to all of length;
    where there are three or more, the last only begins."""
    B, top = case["B"], case["length"]
    if B == 1:
        return [top]
    out = [int(top * (0.25 + 0.75 * ((b * 0.6180339887) % 1.0))) for b in range(B)]
    out[0] = top
    if B >= 3:
        out[-1] = 0
    return out


def _counts(case):
    """Drafted tokens of each sequence in use: up to three fewer than T."""
    return [max(1, case["T"] - b % 4) if case["B"] > 1 else case["T"] for b in range(case["B"])]


def _accepted(case):
    return [1 + (3 + 7 * b) % case["keep"] for b in range(case["B"])]


def _columns(case):
    return (max(_lengths(case)) + case["T"] + case["page"] - 1) // case["page"]


# ---- inputs ----

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, shape, std=1.0, dtype="f32"):
    out = torch.empty(shape, device="cuda", dtype=_DTYPE[dtype])
    flat, step = out.view(-1), 1 << 27
    for i in range(0, flat.numel(), step):  # no f32 copy of a whole cache
        n = min(step, flat.numel() - i)
        flat[i:i + n] = (torch.randn(n, generator=g, device="cuda", dtype=torch.float32) * std).to(out.dtype)
    return out


def _u32(values):
    """Unsigned words in torch's 32-bit integers."""
    return torch.from_numpy(np.ascontiguousarray(values, dtype=np.uint32).view(np.int32)).cuda()


def _pages(case, rng):
    """The page table [B, columns]: pages of the sequences in random order,
    entries past a sequence's end name none; and the number of pages."""
    need = [(n + case["T"] + case["page"] - 1) // case["page"] for n in _lengths(case)]
    pages = sum(need) + 3
    order = rng.permutation(pages)
    table = np.full((case["B"], _columns(case)), _NO_PAGE, np.uint32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def _tree(case, rng):
    """Per row the words of its mask (bit j: it sees drafted token j: its
    ancestors and itself), and its depth."""
    B, T = case["B"], case["T"]
    mask, depth = np.zeros((B, T, (T + 31) // 32 * 4), np.uint8), np.zeros((B, T), np.int64)
    for b in range(B):
        seen = []
        for i in range(T):
            # Often the token before it, else any earlier one.
            parent = i - 1 if not case["tree"] or rng.random() < 0.3 else int(rng.integers(0, i)) if i else -1
            seen.append((seen[parent] if i else 0) | 1 << i)
            depth[b, i] = depth[b, parent] + 1 if i else 0
            mask[b, i] = np.frombuffer(seen[i].to_bytes(mask.shape[2], "little"), np.uint8)
    return mask.view(np.uint32).reshape(B * T, -1), depth


def _inputs(case, seed):
    """The case's inputs as torch tensors."""
    g, rng, kind = _generator(seed), np.random.default_rng(seed), case["kind"]
    if kind == "norm":
        M, width = case["M"], case["width"]
        gate = {None: None, "columns": (width,), "rows": (M, width)}[case["gate"]]
        return {"stream": _normal(g, (M, width), 2.0, case["stream"]),
                "update": _normal(g, (M, width), 0.5, case["update"]),
                "weight": _normal(g, (width,), 0.2, "bf16") + 1,
                "post_weight": _normal(g, (width,), 0.2, "bf16") + 1 if case["post"] else None,
                "gate": _normal(g, gate, 0.5, "bf16") if gate else None}
    table, pages = _pages(case, rng)
    shape = (case.get("layers", 1), pages, case["kv"], case["page"], case["dim"])
    out = {"table": _u32(table), "lengths": _u32(_lengths(case)),
           "counts": _u32(_counts(case)) if kind != "commit" else None,
           "keys": _normal(g, shape, 1.0, case["dtype"]), "values": _normal(g, shape, 1.0, case["dtype"])}
    R = case["B"] * case["T"]
    if kind == "commit":
        # The first drafted token continues the text and is always kept; the
        # others of the path lie further down, level by level.
        path = np.zeros((case["B"], case["keep"]), np.uint32)
        for b in range(case["B"]):
            path[b, 1:] = np.sort(rng.choice(np.arange(case["keep"], case["T"]), case["keep"] - 1, replace=False))
        return out | {"path": _u32(path), "accepted": _u32(_accepted(case))}
    mask, depth = _tree(case, rng)
    if kind == "attention":
        # Attention has peaks: scores of a standard deviation of 2.
        out["query"] = _normal(g, (R, case["heads"] * case["dim"]), 2.0, case["dtype"])
        out["mask"] = _u32(mask) if case["tree"] else None
        return out
    positions = depth + np.array(_lengths(case))[:, None]
    half = case["rotary"] // 2
    angle = np.outer(np.arange(positions.max() + 1), _THETA ** (-np.arange(half) / half))
    out["rotary"] = torch.from_numpy(np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)).cuda()
    out["positions"] = _u32(positions.reshape(-1))
    for name, heads in (("query", case["heads"]), ("key", case["kv"]), ("value", case["kv"])):
        out[name] = _normal(g, (R, heads * case["dim"]), 1.0, case["x"])
    return out


# ---- the framework's side ----

_SESSION = None


def _session():
    """One Session for the process, as a program that serves one GPU keeps."""
    global _SESSION
    if _SESSION is None:
        import affon_amd as A
        _SESSION = A.Session("rocm")
    return _SESSION


def _upload(t, into=None):
    """A Session tensor with a torch tensor's values."""
    from affon_amd import _native
    if t is None:
        return None
    name = {torch.float32: "f32", torch.bfloat16: "bf16", torch.int32: "u32"}[t.dtype]
    out = into if into is not None else _session().empty(name, tuple(t.shape))
    t = t.contiguous()
    torch.cuda.synchronize()
    _native.check(_native.load().affon_rocm_memcpy_d2d(_session()._handle, out.data_ptr, t.data_ptr(),
                                                       t.numel() * t.element_size()), "copy")
    return out


class _Interface:
    """A Session tensor as torch can look at it, without a copy."""

    def __init__(self, tensor):
        self.tensor = tensor
        self.__cuda_array_interface__ = {
            "shape": tensor.shape, "typestr": {"f32": "<f4", "bf16": "<i2"}[tensor.dtype],
            "data": (tensor.data_ptr, False), "version": 2, "strides": None}


def _look(tensor):
    t = torch.as_tensor(_Interface(tensor), device="cuda")
    return t.view(torch.bfloat16) if tensor.dtype == "bf16" else t


def _own_state(case, inputs):
    import affon_amd as A
    kind, s = case["kind"], _session()
    if kind == "norm":
        t = {k: _upload(v) for k, v in inputs.items()}
        outs = (s.empty(case["stream"], inputs["stream"].shape), s.empty(case["out"], inputs["stream"].shape))
        state = {"call": A.residual_norm, "args": (t["stream"], t["update"]),
                 "options": {"weight": t["weight"], "post_norm": case["post"], "post_weight": t["post_weight"],
                             "gate": t["gate"], "scale": case["scale"], "epsilon": _EPSILON, "out": outs}}
        return state | {"outputs": [_look(o) for o in outs]}
    layers, pages, kv, page, dim = inputs["keys"].shape
    cache = A.PagedCache(s, layers=layers, pages=pages, kv_heads=kv, page_size=page, head_dim=dim, dtype=case["dtype"])
    _upload(inputs.pop("keys"), cache.keys)
    _upload(inputs.pop("values"), cache.values)
    t = {k: _upload(v) for k, v in inputs.items()}
    batch = A.DraftBatch(t["table"], t["lengths"], rows=case["T"], counts=t["counts"])
    caches = [_look(cache.keys), _look(cache.values)]
    if kind == "commit":
        return {"call": A.cache_commit, "args": (cache, batch, t["path"], t["accepted"]), "options": {},
                "outputs": caches}
    out = s.empty(case["dtype"], inputs["query"].shape)
    if kind == "attention":
        return {"call": A.tree_attention, "args": (cache, batch, t["query"], t["mask"]), "options": {"out": out},
                "outputs": _look(out)}
    return {"call": A.cache_append, "args": (cache, batch, t["query"], t["key"], t["value"], t["positions"], t["rotary"]),
            "options": {"interleaved": case["interleaved"], "out": out}, "outputs": [_look(out), *caches]}


def prepare(case, seed):
    inputs = _inputs(case, seed)
    if own:
        state = _own_state(case, inputs)
        torch.cuda.synchronize()
        return state
    plain = {"norm": _plain_norm, "attention": _plain_attention, "append": _plain_append, "commit": _plain_commit}
    if case["kind"] != "norm":
        inputs["host"] = (_lengths(case), _counts(case))
    return {"call": plain[case["kind"]], "args": (case, inputs), "options": {}, "outputs": None}


def run(state):
    result = state["call"](*state["args"], **state["options"])
    return result if state["outputs"] is None else state["outputs"]


# ---- the plain forms ----

def _plain_norm(case, t):
    x, u = t["stream"].float(), t["update"].float()
    if case["post"]:
        u = u * (u.square().mean(-1, keepdim=True) + _EPSILON).rsqrt() * t["post_weight"].float()
    if t["gate"] is not None:
        u = u * t["gate"].float()
    x = x + case["scale"] * u
    n = x * (x.square().mean(-1, keepdim=True) + _EPSILON).rsqrt() * t["weight"].float()
    return [x.to(_DTYPE[case["stream"]]), n.to(_DTYPE[case["out"]])]


def _plain_attention(case, t):
    B, T, H, D, P = case["B"], case["T"], case["kv"], case["dim"], case["page"]
    G = case["heads"] // H
    out = torch.zeros((B, T, H, G, D), device="cuda")
    query = t["query"].view(B, T, H, G, D)
    bit = torch.arange(T, device="cuda", dtype=torch.int32)
    for b, (length, count) in enumerate(zip(*t["host"])):
        n = length + count
        index = t["table"][b, :(n + P - 1) // P].long()
        k, v = (t[name][0].index_select(0, index).permute(1, 0, 2, 3).reshape(H, -1, D)[:, :n].float()
                for name in ("keys", "values"))
        if t["mask"] is None:
            seen = bit[:, None] >= bit[None, :count]
        else:
            words = t["mask"].view(B, T, -1)[b]
            seen = (words[:, (bit[:count] // 32).long()] >> (bit[:count] % 32)) & 1 != 0
        q = query[b, :count].permute(1, 0, 2, 3).reshape(H, count * G, D).float()
        s = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(D ** -0.5).view(H, count, G, n)
        s[..., length:].masked_fill_(~seen[:count, None, :], -math.inf)
        top = s.amax(-1, keepdim=True)
        e = (s - top.masked_fill(top == -math.inf, 0.0)).exp_()
        total = e.sum(-1)
        o = torch.matmul(e.view(H, count * G, n), v).view(H, count, G, D)
        out[b, :count] = (o / total.masked_fill(total == 0, 1.0)[..., None]).permute(1, 0, 2, 3)
    return out.view(B * T, -1).to(_DTYPE[case["dtype"]])


def _slots(case, t, at):
    """Page and line of token `at` [B, n] of each sequence."""
    page = torch.gather(t["table"].long(), 1, at // case["page"])
    return page, at % case["page"]


def _plain_append(case, t):
    B, T, D, h = case["B"], case["T"], case["dim"], case["rotary"] // 2
    turn = t["rotary"][t["positions"].long()]
    c, s = turn[:, None, :h], turn[:, None, h:]
    used = torch.arange(T, device="cuda")[None, :] < t["counts"].long()[:, None]

    def rotated(x):
        x = x.view(B * T, -1, D).float()
        if case["interleaved"]:
            a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
            turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
        else:
            a, b = x[..., :h], x[..., h:2 * h]
            turned = torch.cat((a * c - b * s, b * c + a * s), -1)
        return torch.cat((turned, x[..., 2 * h:]), -1)

    query = rotated(t["query"]).masked_fill_(~used.reshape(-1, 1, 1), 0.0).view(B * T, -1).to(_DTYPE[case["dtype"]])
    at = t["lengths"].long()[:, None] + torch.arange(T, device="cuda")
    page, line = (v[used] for v in _slots(case, t, at))
    keep = used.reshape(-1)
    t["keys"][0][page, :, line] = rotated(t["key"])[keep].to(_DTYPE[case["dtype"]])
    t["values"][0][page, :, line] = t["value"].view(B * T, -1, D)[keep].float().to(_DTYPE[case["dtype"]])
    return [query, t["keys"], t["values"]]


def _plain_commit(case, t):
    step = torch.arange(case["keep"], device="cuda")
    kept = step < t["accepted"].long()[:, None]
    start = t["lengths"].long()[:, None]
    page, line = (v[kept] for v in _slots(case, t, start + t["path"].long()))
    to_page, to_line = (v[kept] for v in _slots(case, t, start + step))
    for cache in (t["keys"], t["values"]):
        cache[:, to_page, :, to_line] = cache[:, page, :, line]
    return [t["keys"], t["values"]]


# ---- what the path cannot do without ----

def work(case):
    kind = case["kind"]
    if kind == "norm":
        n = case["M"] * case["width"]
        gate = {None: 0, "columns": 2 * case["width"], "rows": 2 * n}[case["gate"]]
        moved = n * (2 * _BYTES[case["stream"]] + _BYTES[case["update"]] + _BYTES[case["out"]])
        return {"bytes": moved + gate + (4 if case["post"] else 2) * case["width"], "flops": 10 * n}
    B, T, D, e = case["B"], case["T"], case["dim"], _BYTES[case["dtype"]]
    if kind == "commit":
        moved = sum(a - 1 for a in _accepted(case))
        return {"bytes": 4 * moved * case["layers"] * case["kv"] * D * e + 4 * B * (3 + case["keep"]), "flops": 0}
    lengths, counts = _lengths(case), _counts(case)
    if kind == "attention":
        tokens = sum(n + c for n, c in zip(lengths, counts))
        pairs = sum((n + c) * c for n, c in zip(lengths, counts))
        mask = 4 * B * T * ((T + 31) // 32) if case["tree"] else 0
        return {"bytes": 2 * tokens * case["kv"] * D * e + 2 * B * T * case["heads"] * D * e + mask +
                4 * B * (2 + _columns(case)), "flops": 4 * pairs * case["heads"] * D}
    rows = sum(counts)
    width = (case["heads"] + 2 * case["kv"]) * D
    positions = min(rows, max(lengths) + T)
    return {"bytes": rows * width * (_BYTES[case["x"]] + e) + positions * case["rotary"] * 4 + 4 * B * T,
            "flops": 3 * rows * (case["heads"] + case["kv"]) * case["rotary"]}


# ---- the definitions in 64 bits ----

def exact(case, seed):
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "norm":
        def normed(v, w):
            return v / torch.sqrt((v * v).sum(-1, keepdim=True) / case["width"] + _EPSILON) * w.double()
        u = t["update"].double()
        u = normed(u, t["post_weight"]) if case["post"] else u
        y = t["stream"].double() + case["scale"] * u * (1.0 if t["gate"] is None else t["gate"].double())
        return [y, normed(y, t["weight"])]
    B, T, H, D, P = case["B"], case["T"], case["kv"], case["dim"], case["page"]
    table = t["table"].cpu().numpy().view(np.uint32).astype(np.int64)
    lengths = _lengths(case)
    if kind == "commit":
        keys, values = t["keys"].clone(), t["values"].clone()
        path = t["path"].cpu().numpy()
        for b, accepted in enumerate(_accepted(case)):
            for i in range(accepted):
                n, m = lengths[b] + i, lengths[b] + int(path[b, i])
                for new, old in ((keys, t["keys"]), (values, t["values"])):
                    new[:, table[b, n // P], :, n % P] = old[:, table[b, m // P], :, m % P]
        return [keys, values]
    counts = _counts(case)
    if kind == "append":
        keys, values = t["keys"].double(), t["values"].double()
        row = t["positions"].cpu().numpy()
        turn = t["rotary"].double()[torch.from_numpy(row.astype(np.int64)).cuda()]
        turn = torch.complex(turn[:, :case["rotary"] // 2], turn[:, case["rotary"] // 2:])

        def turned(x):
            x, r = x.double().reshape(B * T, -1, D).clone(), case["rotary"]
            first = slice(0, r, 2) if case["interleaved"] else slice(0, r // 2)
            second = slice(1, r, 2) if case["interleaved"] else slice(r // 2, r)
            z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
            x[..., first], x[..., second] = z.real, z.imag
            return x
        q, k, v = turned(t["query"]), turned(t["key"]), t["value"].double().reshape(B * T, H, D)
        for b in range(B):
            q[b * T + counts[b]:(b + 1) * T] = 0.0
            n = np.arange(lengths[b], lengths[b] + counts[b])
            page, line = torch.from_numpy(table[b, n // P]).cuda(), torch.from_numpy(n % P).cuda()
            for h in range(H):
                keys[0, :, h][page, line] = k[b * T:b * T + counts[b], h]
                values[0, :, h][page, line] = v[b * T:b * T + counts[b], h]
        return [q.reshape(B * T, -1), keys, values]
    G = case["heads"] // H
    out = torch.zeros((B * T, case["heads"], D), device="cuda", dtype=torch.float64)
    mask = None if t["mask"] is None else t["mask"].cpu().numpy().view(np.uint8)
    for b in range(B):
        n, c = lengths[b] + counts[b], counts[b]
        seen = np.ones((T, n), bool)
        tail = np.tril(np.ones((T, T), bool)) if mask is None else \
            np.unpackbits(mask[b * T:(b + 1) * T], axis=1, bitorder="little")[:, :T].astype(bool)
        seen[:, lengths[b]:] = tail[:, :c]
        seen = torch.from_numpy(seen[:c]).cuda()
        index = torch.from_numpy(table[b, :(n + P - 1) // P]).cuda()
        for h in range(H):
            k = t["keys"][0, :, h].index_select(0, index).reshape(-1, D)[:n].double()
            v = t["values"][0, :, h].index_select(0, index).reshape(-1, D)[:n].double()
            for g in range(G):
                q = t["query"][b * T:b * T + c, (h * G + g) * D:(h * G + g + 1) * D].double()
                s = torch.where(seen, q @ k.T.contiguous() / math.sqrt(D), -math.inf)
                weight = torch.softmax(s, -1).nan_to_num(0.0)
                out[b * T:b * T + c, h * G + g] = weight @ v
    return out.reshape(B * T, -1)
