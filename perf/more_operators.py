"""More operators of a decoder block over a paged cache, as they are measured:
the append with norms of the query and key heads and with positions of several
axes, attention of sequences that share a prefix, the attention weights that
tokens gather, and the eviction of the tokens that gathered least.

Each of B sequences holds lengths[b] tokens in pages that its row of the page
table names, and T drafted tokens, of which counts[b] are in use. Inputs are
made on the GPU from the seed; lengths and counts follow from the case, so
that its work does.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "bf16": 2}
_EPSILON = 1e-6
_THETA = 500000.0
_NO_PAGE = 0xFFFFFFFF


def listed():
    return [
        # One token of one conversation, query and key heads normed: the f32
        # projections of one row, where latency counts.
        {"name": "append_norm_one_token", "kind": "append", "B": 1, "T": 1, "heads": 32, "kv": 8, "dim": 128,
         "rotary": 128, "length": 777, "page": 16, "interleaved": False, "x": "f32", "dtype": "bf16", "norm": "one",
         "sections": None, "mixed": False},
        # Pieces of 1024 tokens of four prompts through a 70B-shaped block.
        {"name": "append_norm_prompt", "kind": "append", "B": 4, "T": 1024, "heads": 64, "kv": 8, "dim": 128,
         "rotary": 128, "length": 1000, "page": 64, "interleaved": False, "x": "f32", "dtype": "bf16", "norm": "one",
         "sections": None, "mixed": False},
        # Two images of 37 x 37 patches after a text: positions of time, height
        # and width, heads normed.
        {"name": "append_axes_image", "kind": "append", "B": 2, "T": 1369, "heads": 32, "kv": 8, "dim": 128,
         "rotary": 128, "length": 200, "page": 16, "interleaved": False, "x": "bf16", "dtype": "bf16", "norm": "heads",
         "sections": "16 24 24", "mixed": False},
        # Odd sizes in f32: pieces of 50 patches, narrow heads, neighbouring
        # pairs that take the axes in turn, no norms.
        {"name": "append_axes_odd_f32", "kind": "append", "B": 3, "T": 50, "heads": 20, "kv": 4, "dim": 80,
         "rotary": 80, "length": 301, "page": 48, "interleaved": True, "x": "f32", "dtype": "f32", "norm": None,
         "sections": "14 13 13", "mixed": True},
        # Four answers to one prompt of about 1000 tokens that only begin.
        {"name": "shared_small", "kind": "shared", "groups": 1, "per": 4, "T": 1, "heads": 32, "kv": 8, "dim": 128,
         "shared": 1008, "own": 40, "page": 16, "tree": False, "dtype": "bf16"},
        # The largest: 64 conversations after one prompt of 32768 tokens, one
        # token each, a 70B-shaped block.
        {"name": "shared_decode_b64", "kind": "shared", "groups": 1, "per": 64, "T": 1, "heads": 64, "kv": 8, "dim": 128,
         "shared": 32768, "own": 1024, "page": 64, "tree": False, "dtype": "bf16"},
        # Eight samples of each of four prompts, trees of five drafted tokens,
        # narrow heads in f32.
        {"name": "shared_samples_f32", "kind": "shared", "groups": 4, "per": 8, "T": 5, "heads": 20, "kv": 4, "dim": 80,
         "shared": 6000, "own": 301, "page": 48, "tree": True, "dtype": "f32"},
        # What one token of one conversation attends to.
        {"name": "weights_one_token", "kind": "weights", "B": 1, "T": 1, "heads": 32, "kv": 8, "dim": 128,
         "length": 777, "page": 16, "tree": False, "dtype": "bf16"},
        # The same for a decode batch of 32 conversations.
        {"name": "weights_decode_b32", "kind": "weights", "B": 32, "T": 1, "heads": 32, "kv": 8, "dim": 128,
         "length": 4096, "page": 64, "tree": False, "dtype": "bf16"},
        # The last 32 tokens of four long prompts look back over them, before
        # the prompts' caches are cut down.
        {"name": "weights_window", "kind": "weights", "B": 4, "T": 32, "heads": 64, "kv": 8, "dim": 128,
         "length": 16384, "page": 64, "tree": False, "dtype": "bf16"},
        # One conversation's cache of one layer, cut to 1024 tokens of which
        # the last 256 stay whatever they gathered.
        {"name": "evict_one", "kind": "evict", "layers": 1, "B": 1, "kv": 8, "dim": 128, "length": 2000, "keep": 1024,
         "recent": 256, "page": 16, "dtype": "bf16"},
        # Every layer of a 32-layer model for eight conversations.
        {"name": "evict_b8_layers", "kind": "evict", "layers": 32, "B": 8, "kv": 8, "dim": 128, "length": 4096,
         "keep": 1024, "recent": 128, "page": 64, "dtype": "bf16"},
    ]


def _log(rng, low, high, step=1):
    """A multiple of step from low to high, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / step)) * step))


def draw(rng: random.Random):
    kind = rng.choice(["append"] * 3 + ["shared"] * 4 + ["weights"] * 3 + ["evict"] * 2)
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    case = {"kind": kind, "kv": rng.choice([1, 2, 4, 8, 8]), "dim": dim, "dtype": rng.choice(["bf16", "bf16", "f32"]),
            "page": rng.choice([16, 16, 32, 48, 64, 128, 256])}
    if kind == "evict":
        case |= {"layers": rng.choice([1, 2, 8, 32]), "B": _log(rng, 1, 16), "length": _log(rng, 64, 32768)}
        while case["layers"] * case["B"] * case["kv"] * case["length"] * dim * _BYTES[case["dtype"]] > 32 * 8 * 8 * 4096 * 256:
            case["length"] = max(32, case["length"] * 2 // 3)
            case["B"] = max(1, case["B"] * 3 // 4)
        case["keep"] = max(2, int(case["length"] * rng.uniform(0.1, 0.9)))
        return case | {"recent": int(case["keep"] * rng.choice([0.0, 0.1, 0.25, 0.5]))}
    case["heads"] = case["kv"] * rng.choice([1, 2, 4, 4, 5, 8])
    if kind == "append":
        rotary = rng.choice([dim, dim, dim // 2])
        sections, norm = None, rng.choice(["one", "one", "heads", None])
        if norm is None or rng.random() < 0.5:
            half, n = rotary // 2, rng.choice([2, 3, 3, 4])
            cuts = sorted(rng.sample(range(1, half), n - 1))
            sections = " ".join(str(b - a) for a, b in zip([0] + cuts, cuts + [half]))
        case |= {"B": _log(rng, 1, 32), "T": _log(rng, 1, 1500), "x": rng.choice(["f32", "f32", "bf16"]),
                 "rotary": rotary, "length": _log(rng, 1, 1024), "interleaved": rng.random() < 0.3, "norm": norm,
                 "sections": sections, "mixed": sections is not None and rng.random() < 0.4}
        while case["B"] * case["T"] * (case["heads"] + 2 * case["kv"]) * dim > 4 * 1024 * 80 * 128:
            case["T"] = max(1, case["T"] // 2)
            case["B"] = max(1, case["B"] * 3 // 4)
        return case
    case |= {"tree": rng.random() < 0.5}
    if kind == "shared":
        case |= {"groups": rng.choice([1, 1, 1, 2, 5]), "per": _log(rng, 1, 64), "T": _log(rng, 1, 24),
                 "shared": _log(rng, case["page"], 32768, case["page"]), "own": _log(rng, 1, 2048)}
        top, shrink = "shared_decode_b64", ("shared", "per")
    else:
        case |= {"B": _log(rng, 1, 48), "T": _log(rng, 1, 64), "length": _log(rng, 1, 16384)}
        top, shrink = "weights_window", ("length", "B")
    # A listed case bounds it; f32 products run at a sixteenth of bf16's rate.
    top = work(next(c for c in listed() if c["name"] == top))
    least = 1 if case["dtype"] == "bf16" else 16
    while work(case)["bytes"] > top["bytes"] or work(case)["flops"] * least > top["flops"]:
        case[shrink[0]] = max(1, case[shrink[0]] * 2 // 3)
        if kind == "shared":
            case["shared"] = max(case["page"], case["shared"] // case["page"] * case["page"])
        case[shrink[1]] = max(1, case[shrink[1]] * 3 // 4)
        case["T"] = max(1, case["T"] * 3 // 4)
    return case


# ---- what follows from the case alone ----

def _sequences(case):
    return case["groups"] * case["per"] if case["kind"] == "shared" else case["B"]


def _shared(case):
    """Tokens that each group's sequences share, in whole pages."""
    return [max(1, int(case["shared"] * (1 - 0.25 * (g % 3))) // case["page"]) * case["page"]
            for g in range(case["groups"])]


def _lengths(case):
    """Committed tokens of each sequence: from a quarter to all of length (of
    its own ones, where a prefix is shared); where there are three or more, the
    last only begins, but an evicted one."""
    B, top = _sequences(case), case["own"] if case["kind"] == "shared" else case["length"]
    out = [int(top * (0.25 + 0.75 * ((b * 0.6180339887) % 1.0))) for b in range(B)]
    out[0] = top
    if B >= 3 and case["kind"] != "evict":
        out[-1] = 0
    return [n + _shared(case)[b // case["per"]] for b, n in enumerate(out)] if case["kind"] == "shared" else out


def _counts(case):
    """Drafted tokens of each sequence in use: up to three fewer than T."""
    B, T = _sequences(case), case["T"]
    return [max(1, T - b % 4) if B > 1 else T for b in range(B)]


def _columns(case):
    return (max(_lengths(case)) + case.get("T", 0) + case["page"] - 1) // case["page"]


def _kept(case):
    return [min(n, case["keep"]) for n in _lengths(case)]


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
    """The page table [B, columns]: pages of the sequences in random order, a
    group's shared ones in all its rows; entries past a sequence's end name
    none; and the number of pages."""
    P, B = case["page"], _sequences(case)
    need = [(n + case.get("T", 0) + P - 1) // P for n in _lengths(case)]
    before = [_shared(case)[b // case["per"]] // P for b in range(B)] if case["kind"] == "shared" else [0] * B
    first = [b % case["per"] == 0 if case["kind"] == "shared" else True for b in range(B)]
    pages = sum(n if f else n - m for n, m, f in zip(need, before, first)) + 3
    order = rng.permutation(pages)
    table = np.full((B, _columns(case)), _NO_PAGE, np.uint32)
    at = 0
    for b, n in enumerate(need):
        start = 0 if first[b] else before[b]
        if start:
            table[b, :start] = table[b // case["per"] * case["per"], :start]
        table[b, start:n] = order[at:at + n - start]
        at += n - start
    return table, pages


def _tree(case, rng):
    """Per row the words of its mask (bit j: it sees drafted token j: its
    ancestors and itself)."""
    B, T = _sequences(case), case["T"]
    mask = np.zeros((B, T, (T + 31) // 32 * 4), np.uint8)
    for b in range(B):
        seen = []
        for i in range(T):
            # Often the token before it, else any earlier one.
            parent = i - 1 if rng.random() < 0.3 else int(rng.integers(0, i)) if i else -1
            seen.append((seen[parent] if i else 0) | 1 << i)
            mask[b, i] = np.frombuffer(seen[i].to_bytes(mask.shape[2], "little"), np.uint8)
    return mask.view(np.uint32).reshape(B * T, -1)


def _sections(case):
    """Pairs of each axis."""
    return [int(n) for n in case["sections"].split()]


def _positions(case):
    """[axes, B*T]: drafted token i follows its sequence's; with axes, patch i
    of an image of about T patches: time stands still, height and width walk."""
    start = np.array(_lengths(case))[:, None]
    i = np.broadcast_to(np.arange(case["T"]), (case["B"], case["T"]))
    if case["sections"] is None:
        return (start + i).reshape(1, -1)
    side = max(1, math.isqrt(case["T"]))
    axes = [start + 0 * i, start + i // side, start + i % side, start + i % 3]
    return np.stack([a.reshape(-1) for a in axes[:len(_sections(case))]])


def _axes(case):
    """Axis of each pair: the sections one after the other, or the axes in turn
    while each has pairs left."""
    if case["sections"] is None:
        return [0] * (case["rotary"] // 2)
    sections = _sections(case)
    if not case["mixed"]:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [a for turn in range(max(sections)) for a, n in enumerate(sections) if turn < n]


def _inputs(case, seed):
    """The case's inputs as torch tensors."""
    g, rng, kind = _generator(seed), np.random.default_rng(seed), case["kind"]
    table, pages = _pages(case, rng)
    shape = (case.get("layers", 1), pages, case["kv"], case["page"], case["dim"])
    out = {"table": _u32(table), "lengths": _u32(_lengths(case)),
           "keys": _normal(g, shape, 1.0, case["dtype"])}
    if kind != "weights":  # the weights come from the keys alone
        out["values"] = _normal(g, shape, 1.0, case["dtype"])
    B, D = _sequences(case), case["dim"]
    gathered = (case.get("layers", 1), B, case["kv"], _columns(case) * case["page"])
    if kind == "evict":
        # A few tokens gather most; some have gathered nothing yet.
        weights = torch.exp(_normal(g, gathered, 2.0))
        out["weights"] = weights * (torch.rand(gathered, generator=g, device="cuda") > 0.1)
        return out | {"keep": _u32([case["keep"]] * B), "recent": _u32([case["recent"]] * B)}
    out["counts"] = _u32(_counts(case))
    R = B * case["T"]
    if kind != "append":
        # Attention has peaks: scores of a standard deviation of 2.
        out["query"] = _normal(g, (R, case["heads"] * D), 2.0, case["dtype"])
        out["mask"] = _u32(_tree(case, rng)) if case["tree"] else None
        if kind == "shared":
            return out | {"shared": _u32(_shared(case))}
        # What a few calls before gathered: a row's and head's weights sum to 1.
        each = case["T"] * case["heads"] / case["kv"] / case["length"]
        return out | {"weights": torch.exp(_normal(g, gathered, 1.0)) * each}
    positions = _positions(case)
    half = case["rotary"] // 2
    angle = np.outer(np.arange(positions.max() + 1), _THETA ** (-np.arange(half) / half))
    out["rotary"] = torch.from_numpy(np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)).cuda()
    out["positions"] = _u32(positions)
    for name, heads in (("query", case["heads"]), ("key", case["kv"]), ("value", case["kv"])):
        out[name] = _normal(g, (R, heads * D), 1.5, case["x"])
    for name, heads in (("query_norm", case["heads"]), ("key_norm", case["kv"])):
        shape = {"one": (D,), "heads": (heads * D,), None: None}[case["norm"]]
        out[name] = _normal(g, shape, 0.2, "bf16") + 1 if shape else None
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
    layers, pages, kv, page, dim = inputs["keys"].shape
    cache = A.PagedCache(s, layers=layers, pages=pages, kv_heads=kv, page_size=page, head_dim=dim, dtype=case["dtype"])
    _upload(inputs.pop("keys"), cache.keys)
    if "values" in inputs:
        _upload(inputs.pop("values"), cache.values)
    t = {k: _upload(v) for k, v in inputs.items()}
    batch = A.DraftBatch(t["table"], t["lengths"], rows=case.get("T", 1), counts=t.get("counts"))
    caches = [_look(cache.keys), _look(cache.values)]
    if kind == "evict":
        out = s.empty("f32", inputs["weights"].shape)
        return {"call": A.cache_evict, "args": (cache, batch, t["weights"], t["keep"], t["recent"]),
                "options": {"out": out}, "outputs": [_look(out), *caches]}
    if kind == "weights":
        return {"call": A.attention_weights, "args": (cache, batch, t["query"], t["weights"], t["mask"]), "options": {},
                "outputs": _look(t["weights"])}
    out = s.empty(case["dtype"], inputs["query"].shape)
    if kind == "shared":
        return {"call": A.shared_attention, "args": (cache, batch, t["query"], t["shared"], t["mask"]),
                "options": {"out": out}, "outputs": _look(out)}
    options = {"interleaved": case["interleaved"], "query_norm": t["query_norm"], "key_norm": t["key_norm"],
               "epsilon": _EPSILON, "out": out}
    if case["sections"] is not None:
        options["axes"] = A.rotary_axes(_sections(case), interleaved=case["mixed"])
    else:
        t["positions"] = _upload(inputs["positions"].view(-1))
    return {"call": A.cache_append, "args": (cache, batch, t["query"], t["key"], t["value"], t["positions"], t["rotary"]),
            "options": options, "outputs": [_look(out), *caches]}


def prepare(case, seed):
    inputs = _inputs(case, seed)
    if own:
        state = _own_state(case, inputs)
        torch.cuda.synchronize()
        return state
    plain = {"append": _plain_append, "shared": _plain_shared, "weights": _plain_weights, "evict": _plain_evict}
    return {"call": plain[case["kind"]], "args": (case, inputs), "options": {}, "outputs": None}


def run(state):
    result = state["call"](*state["args"], **state["options"])
    return result if state["outputs"] is None else state["outputs"]


# ---- the plain forms ----

def _slots(case, table, at):
    """Page and line of token `at` [R, n] of each row of the table."""
    page = torch.gather(table.long(), 1, at // case["page"])
    return page, at % case["page"]


def _lines(case, t, name, table, at):
    """Keys or values [R, kv, n, dim] in f32 of tokens `at` [R, n]; tokens that lie nowhere give some page's."""
    page, line = _slots(case, table, at)
    pages = t[name].shape[1]
    return t[name][0][torch.where((page >= 0) & (page < pages), page, 0), :, line].permute(0, 2, 1, 3).float()


def _used(case, t, B):
    return torch.arange(case["T"], device="cuda")[None, :] < t["counts"].long()[:, None]


def _plain_append(case, t):
    B, T, D, h = case["B"], case["T"], case["dim"], case["rotary"] // 2
    axis = torch.tensor(_axes(case), device="cuda")
    place = t["positions"].long()[axis].T  # of each row's pairs
    pair = torch.arange(h, device="cuda")
    c, s = t["rotary"][place, pair][:, None], t["rotary"][place, h + pair][:, None]
    used = _used(case, t, B)

    def rotated(x, weight):
        x = x.view(B * T, -1, D).float()
        if weight is not None:
            x = x * (x.square().mean(-1, keepdim=True) + _EPSILON).rsqrt() * weight.float().view(-1, D)
        if case["interleaved"]:
            a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
            turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
        else:
            a, b = x[..., :h], x[..., h:2 * h]
            turned = torch.cat((a * c - b * s, b * c + a * s), -1)
        return torch.cat((turned, x[..., 2 * h:]), -1)

    query = rotated(t["query"], t["query_norm"]).masked_fill_(~used.reshape(-1, 1, 1), 0.0)
    at = t["lengths"].long()[:, None] + torch.arange(T, device="cuda")
    page, line = (v[used] for v in _slots(case, t["table"], at))
    keep = used.reshape(-1)
    t["keys"][0][page, :, line] = rotated(t["key"], t["key_norm"])[keep].to(_DTYPE[case["dtype"]])
    t["values"][0][page, :, line] = t["value"].view(B * T, -1, D)[keep].float().to(_DTYPE[case["dtype"]])
    return [query.view(B * T, -1).to(_DTYPE[case["dtype"]]), t["keys"], t["values"]]


def _seen(case, t, start, n):
    """Which of its tokens start[b] .. start[b] + n - 1 row (b, i) sees, bool [B, T, n]."""
    B, T = _sequences(case), case["T"]
    at = start[:, None] + torch.arange(n, device="cuda") - t["lengths"].long()[:, None]  # of the drafted ones
    row = torch.arange(T, device="cuda")
    j = at.clamp(0, T - 1)
    if t["mask"] is None:
        drafted = j[:, None, :] <= row[None, :, None]
    else:
        words = t["mask"].view(B, T, -1)
        word = torch.gather(words, 2, (j // 32)[:, None, :].expand(B, T, n))
        drafted = (word >> (j % 32)[:, None, :].int()) & 1 != 0
    counts = t["counts"].long()[:, None, None]
    drafted = drafted & (at[:, None, :] < counts)
    return torch.where(at[:, None, :] < 0, True, drafted) & (row[None, :, None] < counts)


def _plain_shared(case, t):
    groups, per, T, H, D = case["groups"], case["per"], case["T"], case["kv"], case["dim"]
    B, G = groups * per, case["heads"] // H
    query = t["query"].float().view(groups, per * T, H, G, D).permute(0, 2, 1, 3, 4).reshape(groups * H, per * T * G, D)
    shared = t["shared"].long()
    S, O = max(_shared(case)), max(n - _shared(case)[b // per] for b, n in enumerate(_lengths(case))) + T
    at = torch.arange(S, device="cuda")
    place = at.expand(groups, S)
    k, v = (_lines(case, t, name, t["table"].view(groups, per, -1)[:, 0], place).reshape(groups * H, S, D)
            for name in ("keys", "values"))
    first = torch.matmul(query, k.transpose(1, 2).contiguous()).mul_(D ** -0.5).view(groups, H, per * T * G, S)
    first.masked_fill_((at >= shared[:, None])[:, None, None, :], -math.inf)
    # The own tokens of each sequence, after its group's.
    start = shared.repeat_interleave(per)
    place = (start[:, None] + torch.arange(O, device="cuda")).clamp(max=t["table"].shape[1] * case["page"] - 1)
    ok, ov = (_lines(case, t, name, t["table"], place).reshape(B * H, O, D) for name in ("keys", "values"))
    oq = query.view(groups, H, per, T * G, D).transpose(1, 2).reshape(B * H, T * G, D)
    then = torch.matmul(oq, ok.transpose(1, 2).contiguous()).mul_(D ** -0.5).view(B, H, T, G, O)
    then.masked_fill_(~_seen(case, t, start, O)[:, None, :, None, :], -math.inf)
    then = then.view(groups, per, H, T * G, O).transpose(1, 2).reshape(groups, H, per * T * G, O)
    top = torch.maximum(first.amax(-1, keepdim=True), then.amax(-1, keepdim=True))
    first, then = (first - top).exp_(), (then - top).exp_()
    total = first.sum(-1) + then.sum(-1)
    o = torch.matmul(first.view(groups * H, -1, S), v).view(groups, H, per, T * G, D)
    then = then.view(groups, H, per, T * G, O).transpose(1, 2).reshape(B * H, T * G, O)
    o = o + torch.matmul(then, ov).view(groups, per, H, T * G, D).transpose(1, 2)
    o = (o / total.view(groups, H, per, T * G, 1)).view(groups, H, per, T, G, D).permute(0, 2, 3, 1, 4, 5)
    o = o.reshape(B, T, -1).masked_fill(~_used(case, t, B)[..., None], 0.0)
    return o.view(B * T, -1).to(_DTYPE[case["dtype"]])


def _plain_weights(case, t):
    B, T, H, D = case["B"], case["T"], case["kv"], case["dim"]
    G, n = case["heads"] // H, t["weights"].shape[-1]
    at = torch.arange(n, device="cuda").expand(B, n)
    k = _lines(case, t, "keys", t["table"], at).reshape(B * H, n, D)
    q = t["query"].float().view(B, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(B * H, T * G, D)
    s = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(D ** -0.5).view(B, H, T, G, n)
    seen = _seen(case, t, torch.zeros_like(t["lengths"].long()), n)[:, None, :, None, :]
    s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = (s - top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = e.sum(-1, keepdim=True)
    gathered = (e / total.masked_fill(total == 0, 1.0)).sum((2, 3))
    # Added to what committed tokens gathered before; drafted ones begin.
    length, count = t["lengths"].long()[:, None, None], t["counts"].long()[:, None, None]
    w = t["weights"][0]
    w.copy_(torch.where(at[:, None] < length, w + gathered, torch.where(at[:, None] < length + count, gathered, w)))
    return t["weights"]


def _plain_evict(case, t):
    w, D = t["weights"], case["dim"]
    L, B, H, n = w.shape
    at = torch.arange(n, device="cuda")
    length, keep, recent = (t[name].long()[None, :, None, None] for name in ("lengths", "keep", "recent"))
    left = torch.minimum(length, keep)  # tokens afterwards
    last = at >= length - torch.minimum(recent, left)
    score = w.masked_fill(last, -1.0)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, at.expand_as(order))
    kept = (at < length) & (last | (rank < left - torch.minimum(recent, left)))
    source = torch.sort(torch.where(kept, at, n), dim=-1).values  # kept tokens in their order, then n
    there = source < n
    out = torch.where(there, torch.gather(w, -1, source.clamp(max=n - 1)), 0.0)
    layer, b, h, to = there.nonzero(as_tuple=True)
    place = source[layer, b, h, to]
    table, P = t["table"].long(), case["page"]
    for cache in (t["keys"], t["values"]):
        cache[layer, table[b, to // P], h, to % P] = cache[layer, table[b, place // P], h, place % P]
    return [out, t["keys"], t["values"]]


# ---- what the path cannot do without ----

def work(case):
    kind, D, e = case["kind"], case["dim"], _BYTES[case["dtype"]]
    lengths, columns = _lengths(case), _columns(case)
    if kind == "evict":
        rows = case["layers"] * case["kv"]
        moved = sum(k for n, k in zip(lengths, _kept(case)) if k < n)
        return {"bytes": rows * (4 * sum(lengths) + 4 * len(lengths) * columns * case["page"] + 4 * moved * D * e) +
                4 * len(lengths) * (3 + columns), "flops": rows * sum(lengths)}
    B, T, counts = _sequences(case), case["T"], _counts(case)
    tables = 4 * B * (2 + columns)
    if kind == "append":
        rows = sum(counts)
        width = (case["heads"] + 2 * case["kv"]) * D
        positions = min(rows, max(lengths) + T)
        norms = {None: 0, "one": 4 * D, "heads": 2 * (case["heads"] + case["kv"]) * D}[case["norm"]]
        turned = rows * (case["heads"] + case["kv"])
        return {"bytes": rows * width * (_BYTES[case["x"]] + e) + positions * case["rotary"] * 4 + norms +
                4 * B * T * (len(_sections(case)) if case["sections"] else 1),
                "flops": 3 * turned * case["rotary"] + (4 * turned * D if case["norm"] else 0)}
    pairs = sum((n + c) * c for n, c in zip(lengths, counts))
    mask = 4 * B * T * ((T + 31) // 32) if case["tree"] else 0
    if kind == "weights":
        tokens = sum(n + c for n, c in zip(lengths, counts))
        return {"bytes": tokens * case["kv"] * (D * e + 8) + B * T * case["heads"] * D * e + mask + tables,
                "flops": 2 * pairs * case["heads"] * D}
    tokens = sum(_shared(case)) + sum(n + c - _shared(case)[b // case["per"]]
                                      for b, (n, c) in enumerate(zip(lengths, counts)))
    return {"bytes": 2 * tokens * case["kv"] * D * e + 2 * B * T * case["heads"] * D * e + mask + tables,
            "flops": 4 * pairs * case["heads"] * D}


# ---- the definitions in 64 bits ----

def _attended(case, t, name, table, b, h, n):
    """Keys or values [n, D] of head h of sequence b in f64."""
    at = np.arange(n)
    page = torch.from_numpy(table[b, at // case["page"]]).cuda()
    return t[name][0, page, h, torch.from_numpy(at % case["page"]).cuda()].double()


def exact(case, seed):
    t, kind, D, P = _inputs(case, seed), case["kind"], case["dim"], case["page"]
    table = t["table"].cpu().numpy().view(np.uint32).astype(np.int64)
    lengths = _lengths(case)
    if kind == "evict":
        weights = t["weights"].cpu().numpy().astype(np.float64)
        keys, values, out = t["keys"].double(), t["values"].double(), np.zeros_like(weights)
        for layer, b, h in np.ndindex(*weights.shape[:3]):
            n, row = lengths[b], weights[layer, b, h]
            left = min(n, case["keep"])
            recent = min(case["recent"], left)
            best = np.lexsort((np.arange(n - recent), -row[:n - recent]))[:left - recent]
            kept = np.concatenate([np.sort(best), np.arange(n - recent, n)]).astype(np.int64)
            out[layer, b, h, :left] = row[kept]
            to = np.arange(left)
            for new, old in ((keys, t["keys"]), (values, t["values"])):
                moved = old[layer, torch.from_numpy(table[b, kept // P]).cuda(), h, torch.from_numpy(kept % P).cuda()]
                new[layer, torch.from_numpy(table[b, to // P]).cuda(), h, torch.from_numpy(to % P).cuda()] = moved.double()
        return [torch.from_numpy(out).cuda(), keys, values]
    B, T, H, counts = _sequences(case), case["T"], case["kv"], _counts(case)
    if kind == "append":
        keys, values = t["keys"].double(), t["values"].double()
        positions, half = _positions(case), case["rotary"] // 2
        turn = np.zeros((B * T, half), np.int64)
        for j, axis in enumerate(_axes(case)):
            turn[:, j] = positions[axis]
        turn, pair = torch.from_numpy(turn).cuda(), torch.arange(half, device="cuda")
        turn = torch.complex(t["rotary"].double()[turn, pair], t["rotary"].double()[turn, half + pair])

        def turned(x, weight):
            x, r = x.double().reshape(B * T, -1, D).clone(), case["rotary"]
            if weight is not None:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + _EPSILON) * weight.double().reshape(-1, D)
            first = slice(0, r, 2) if case["interleaved"] else slice(0, r // 2)
            second = slice(1, r, 2) if case["interleaved"] else slice(r // 2, r)
            z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
            x[..., first], x[..., second] = z.real, z.imag
            return x
        q, k = turned(t["query"], t["query_norm"]), turned(t["key"], t["key_norm"])
        v = t["value"].double().reshape(B * T, H, D)
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
    gathered = t["weights"].double() if kind == "weights" else None
    mask = None if t["mask"] is None else t["mask"].cpu().numpy().view(np.uint8)
    for b in range(B):
        n, c = lengths[b] + counts[b], counts[b]
        seen = np.ones((T, n), bool)
        tail = np.tril(np.ones((T, T), bool)) if mask is None else \
            np.unpackbits(mask[b * T:(b + 1) * T], axis=1, bitorder="little")[:, :T].astype(bool)
        seen[:, lengths[b]:] = tail[:, :c]
        seen = torch.from_numpy(seen[:c]).cuda()
        for h in range(H):
            k = _attended(case, t, "keys", table, b, h, n).T.contiguous()
            total = torch.zeros(n, device="cuda", dtype=torch.float64)
            if kind == "shared":
                v = _attended(case, t, "values", table, b, h, n)
            for g in range(G):
                q = t["query"][b * T:b * T + c, (h * G + g) * D:(h * G + g + 1) * D].double()
                s = torch.where(seen, q @ k / math.sqrt(D), -math.inf)
                weight = torch.softmax(s, -1).nan_to_num(0.0)
                if kind == "shared":
                    out[b * T:b * T + c, h * G + g] = weight @ v
                else:
                    total += weight.sum(0)
            if kind == "weights":
                gathered[0, b, h, :lengths[b]] += total[:lengths[b]]
                gathered[0, b, h, lengths[b]:n] = total[lengths[b]:]
    return gathered if kind == "weights" else out.reshape(B * T, -1)
