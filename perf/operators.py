"""The operators of a served transformer's step -- rotary positions, the paged key-value cache's
append, one-token attention over that cache, and products with 4-bit weights -- as cases with real
sizes, each in a plain form of elementary torch operations and, with ``own`` set, as the calls of
``cmpext3.ops``."""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DTYPE = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
_SIZE = {"bfloat16": 2, "float16": 2, "float32": 4}
_ROPE_BASE = 10000.0


def _ops():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-cmp-patch_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    os.environ.setdefault("CMPEXT3_AUTOPATCH", "0")
    import cmpext3
    return cmpext3.ops


# -------------------------------------------------------------------------------------------------
# cases
# -------------------------------------------------------------------------------------------------

def _attention(batch, heads, heads_kv, dim, page, longest, shortest, dtype):
    return {"op": "paged_attention", "batch": batch, "heads": heads, "heads_kv": heads_kv, "dim": dim,
            "page": page, "longest": longest, "shortest": shortest, "dtype": dtype}


def _append(batch, heads, heads_kv, dim, page, tokens, past, rot, axes, interleaved, dtype):
    return {"op": "kv_append", "batch": batch, "heads": heads, "heads_kv": heads_kv, "dim": dim, "page": page,
            "tokens": tokens, "past": past, "rot": rot, "axes": axes, "interleaved": interleaved, "dtype": dtype}


def _rope(batch, heads, length, dim, rot, axes, interleaved, grad, dtype):
    return {"op": "rope", "batch": batch, "heads": heads, "length": length, "dim": dim, "rot": rot, "axes": axes,
            "interleaved": interleaved, "grad": grad, "dtype": dtype}


def _linear(tokens, n, k, group, zeros, bias, dtype):
    return {"op": "linear_w4", "tokens": tokens, "n": n, "k": k, "group": group, "zeros": zeros, "bias": bias,
            "dtype": dtype}


def listed():
    named = [
        # one chat turn's first tokens: everything is latency
        ("attention short", _attention(1, 8, 2, 64, 16, 130, 130, "float16")),
        # a serving batch of the 32-head, 128-wide causal model: sequences of every age, one just
        # admitted and one empty slot
        ("attention batch", _attention(32, 32, 8, 128, 64, 8192, 64, "bfloat16")),
        # one document-sized context, which only a split over its length spreads over the GPU
        ("attention long", _attention(1, 32, 8, 128, 16, 131072, 131072, "bfloat16")),
        # full precision, one head per key head, a head of 40 and pages that end inside a tile
        ("attention fp32", _attention(4, 8, 8, 40, 24, 4096, 100, "float32")),
        # one decoding step of the serving batch: query and key rotated, key and value stored
        ("append step", _append(64, 32, 8, 128, 64, 1, 256, 128, 1, False, "bfloat16")),
        # prompts of different lengths admitted together, padded to the longest
        ("append prompts", _append(4, 16, 16, 64, 16, 2048, 0, 64, 1, True, "float16")),
        # text tokens of an image model's cross attention
        ("rope short", _rope(1, 10, 77, 64, 64, 1, False, False, "float16")),
        # video latents: time, height and width each turn a section of the head
        ("rope video", _rope(2, 32, 8192, 128, 128, 3, False, False, "bfloat16")),
        # a training step of an image model in full precision: two axes, part of the head turned
        ("rope training", _rope(2, 8, 4096, 40, 32, 2, True, True, "float32")),
        # one token through a square projection
        ("linear one token", _linear(1, 4096, 4096, 128, False, False, "bfloat16")),
        # eight sequences through the widening projection, zero points stored
        ("linear eight tokens", _linear(8, 16384, 4096, 64, True, True, "float16")),
        # full-precision activations, small groups, odd rows
        ("linear fp32", _linear(3, 1001, 2560, 32, True, True, "float32")),
    ]
    return [dict(case, name=name) for name, case in named]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["paged_attention", "kv_append", "rope", "linear_w4"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    size = _SIZE[dtype]
    dim = rng.choice([40, 64, 80, 96, 128, 128, 160, 192, 256])
    rot = rng.choice([dim, dim, dim // 4 * 2, 32])
    axes = rng.choice([1, 1, 2, 3])
    if op == "paged_attention":
        heads_kv = rng.choice([1, 2, 3, 4, 8, 16])
        batch = _spread(rng, 1, 64)
        room = 5.3e8 / (2 * batch * heads_kv * dim * size)
        longest = _spread(rng, 1, max(1, min(65536, int(room))))
        return _attention(batch, heads_kv * rng.choice([1, 2, 4, 5, 8, 16]), heads_kv, dim,
                          rng.choice([8, 16, 24, 32, 64, 100, 128, 256]), longest, rng.choice([1, longest, (longest + 9) // 10]),
                          dtype)
    if op == "kv_append":
        heads_kv = rng.choice([1, 2, 3, 4, 8, 16])
        heads = heads_kv * rng.choice([0, 1, 4, 5, 8])
        batch = _spread(rng, 1, 64)
        tokens = rng.choice([1, _spread(rng, 2, max(2, min(2048, int(2e8 / (batch * (heads + heads_kv) * dim * size)))))])
        past = _spread(rng, 1, 16384 // batch + 64)
        return _append(batch, heads, heads_kv, dim, rng.choice([8, 16, 24, 32, 64, 100, 128, 256]), tokens, past, rot, axes,
                       rng.random() < 0.5, dtype)
    if op == "rope":
        batch, heads = _spread(rng, 1, 4), rng.choice([1, 5, 8, 10, 16, 32])
        grad = rng.random() < 0.4
        room = 1.3e8 / (batch * heads * dim * size * (2 if grad else 1))
        return _rope(batch, heads, _spread(rng, 1, min(16384, int(room))), dim, rot, axes, rng.random() < 0.5, grad, dtype)
    group = rng.choice([32, 64, 128])
    k = group * _spread(rng, 1, 16384 // group)
    return _linear(_spread(rng, 1, 16), _spread(rng, 1, min(16384, 2**26 // k)), k, group, rng.random() < 0.5,
                   rng.random() < 0.5, dtype)


def _lengths(case):
    """The sequences' lengths: steps of one ratio from the shortest to the longest; in a batch of
    four and more one sequence is empty and one has a single token."""
    n, lo, hi = case["batch"], case["shortest"], case["longest"]
    out = [hi if n == 1 else round(lo * (hi / lo) ** (i / (n - 1))) for i in range(n)]
    if n >= 4 and lo < hi:
        out[0], out[1] = 0, 1
    return out


def _new_lengths(case):
    """Tokens that each sequence appends: all of them in a decoding step; prompts end at different
    places and one in four batch rows is padding to its end."""
    n, length = case["batch"], case["tokens"]
    if length == 1:
        return [1] * n
    return [length - (i * length) // n if i % 4 != 3 else 0 for i in range(n)]


def _sections(rot, axes):
    pairs = rot // 2
    if axes == 1:
        return None
    if axes == 2:
        return (pairs // 2, pairs - pairs // 2)
    side = pairs * 3 // 8
    return (pairs - 2 * side, side, side)


def _grid(tokens, axes, start, device):
    """[axes, batch, tokens] whole coordinates of tokens on a grid that begins at start[batch]."""
    i = torch.arange(tokens, device=device)
    side = max(1, round(tokens ** (1 / axes)))
    place = [i // side ** (axes - 1 - a) % (side if a else 2**31) for a in range(axes)]
    return (torch.stack(place)[:, None, :] + start[None, :, None]).to(torch.int32)


# -------------------------------------------------------------------------------------------------
# inputs
# -------------------------------------------------------------------------------------------------

def _paged(case, needed, gen, device):
    """Caches [pages, heads_kv, page, dim] filled with keys and values, and a page table whose pages
    lie anywhere in them; entries behind a sequence's last page hold -1."""
    page = case["page"]
    counts = [-(-n // page) for n in needed]
    pool = sum(counts) + 3
    order = torch.randperm(pool, generator=gen, device=device).to(torch.int32)
    table = torch.full((len(needed), max(1, max(counts))), -1, dtype=torch.int32, device=device)
    at = 0
    for row, c in enumerate(counts):
        table[row, :c] = order[at:at + c]
        at += c
    shape = (pool, case["heads_kv"], page, case["dim"])
    k, v = (torch.randn(shape, generator=gen, device=device, dtype=_DTYPE[case["dtype"]]) for _ in range(2))
    return {"k_cache": k, "v_cache": v, "page_table": table}


def _turning(case, device):
    """The frequency of every pair, the pairs of each axis, and the axis of every pair."""
    rot, sections = case["rot"], _sections(case["rot"], case["axes"])
    j = torch.arange(rot // 2, device=device, dtype=torch.float64)
    axis = None if sections is None else torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=device)
    return {"freqs": (_ROPE_BASE ** (-2.0 * j / rot)).float(), "sections": sections, "axis": axis}


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = _DTYPE[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=device, dtype=dtype)

    state = {"case": case}
    if case["op"] == "paged_attention":
        turn = seed % case["batch"]
        lengths = _lengths(case)
        lengths = lengths[turn:] + lengths[:turn]
        state |= _paged(case, lengths, gen, device)
        state["query"] = randn(case["batch"], case["heads"], 1, case["dim"])
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=device)
    elif case["op"] == "kv_append":
        turn = seed % case["batch"]
        new = _new_lengths(case)
        new = new[turn:] + new[:turn]
        past = [case["past"] * (i + 1) // case["batch"] for i in range(case["batch"])]
        total = [p + n for p, n in zip(past, new)]
        state |= _paged(case, total, gen, device)
        b, t, d = case["batch"], case["tokens"], case["dim"]
        # as a projection leaves them: [batch, tokens, heads, dim], seen as [batch, heads, tokens, dim]
        state["key"], state["value"] = (randn(b, t, case["heads_kv"], d).transpose(1, 2) for _ in range(2))
        state["query"] = randn(b, t, case["heads"], d).transpose(1, 2) if case["heads"] else None
        state["lengths"] = torch.tensor(total, dtype=torch.int32, device=device)
        state["new_lengths"] = None if t == 1 else torch.tensor(new, dtype=torch.int32, device=device)
        state |= _turning(case, device)
        start = torch.tensor(past, device=device)
        state["positions"] = None if case["axes"] == 1 else _grid(t, case["axes"], start, device)
    elif case["op"] == "rope":
        b, h, n, d = case["batch"], case["heads"], case["length"], case["dim"]
        state["input"] = randn(b, h, n, d).requires_grad_(case["grad"])
        state["grad"] = randn(b, h, n, d) if case["grad"] else None
        state |= _turning(case, device)
        start = torch.randint(0, 100000 if case["axes"] == 1 else 100, (b,), generator=gen, device=device)
        grid = _grid(n, case["axes"], start, device)
        state["positions"] = grid[0] if case["axes"] == 1 else grid
    else:
        m, n, k, group = case["tokens"], case["n"], case["k"], case["group"]
        state["input"] = randn(m, k)
        state["weight"] = torch.randint(0, 256, (n, k // 2), generator=gen, device=device, dtype=torch.uint8)
        scales = torch.rand(n, k // group, generator=gen, device=device) * 0.01 + 0.002
        state["scales"] = scales.to(dtype)
        state["zeros"] = (torch.randint(0, 16, (n, k // group), generator=gen, device=device, dtype=torch.uint8)
                          if case["zeros"] else None)
        state["bias"] = randn(n) if case["bias"] else None
    if own:
        state["ops"] = _ops()
    return state


# -------------------------------------------------------------------------------------------------
# one pass
# -------------------------------------------------------------------------------------------------

def _angles(positions, freqs, axis):
    """cos and sin [batch, 1, tokens, pairs]; positions [batch, tokens], or [axes, batch, tokens]
    with the axis of every pair.  The angles of far positions need 64 bits."""
    place = positions[:, :, None].double() if axis is None else positions[axis].permute(1, 2, 0).double()
    angle = place * freqs.double()
    return torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]


def _rotated(x, cos, sin, interleaved):
    """x [batch, heads, tokens, dim] in 32 bits with its first 2 * pairs values turned."""
    x, pairs = x.float(), cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, x[..., 2 * pairs:]), -1)


def _plain_attention(s):
    q, table = s["query"].float(), s["page_table"].clamp(min=0).long()
    b, h, _, d = q.shape
    hk = s["k_cache"].shape[1]
    # [batch, pages, heads_kv, page, dim] -> [batch, heads_kv, keys, dim]
    k, v = (c[table].float().transpose(1, 2).reshape(b, hk, -1, d) for c in (s["k_cache"], s["v_cache"]))
    scores = q.reshape(b, hk, h // hk, d) @ k.transpose(2, 3) / math.sqrt(d)
    there = (torch.arange(k.shape[2], device=q.device) < s["lengths"][:, None])[:, None, None]
    scores = scores.masked_fill(~there, float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    out = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-38)
    return out.reshape(b, h, 1, d).to(s["query"].dtype)


def _plain_append(s):
    key, value, query, lengths = s["key"], s["value"], s["query"], s["lengths"].long()
    b, hk, t, d = key.shape
    page = s["k_cache"].shape[2]
    token = torch.arange(t, device=key.device)
    new = torch.full_like(lengths, t) if s["new_lengths"] is None else s["new_lengths"].long()
    there = token < new[:, None]
    place = (lengths - new)[:, None] + token
    positions = place if s["positions"] is None else s["positions"]
    cos, sin = _angles(positions, s["freqs"], s["axis"])
    turned = _rotated(key, cos, sin, s["case"]["interleaved"]).to(key.dtype)
    # padding rows store what the first row that is there stores once more
    row = torch.arange(b * t, device=key.device)
    row = torch.where(there.flatten(), row, there.flatten().int().argmax())
    at = place.flatten()[row]
    pages = s["page_table"].long()[row // t, at // page]
    index = (pages[:, None], torch.arange(hk, device=key.device)[None], (at % page)[:, None])
    s["k_cache"][index] = turned.transpose(1, 2).reshape(b * t, hk, d)[row]
    s["v_cache"][index] = value.transpose(1, 2).reshape(b * t, hk, d)[row]
    out = [s["k_cache"], s["v_cache"]]
    if query is not None:
        turned = _rotated(query, cos, sin, s["case"]["interleaved"]).to(query.dtype)
        out.append(torch.where(there[:, None, :, None], turned, query))
    return out


def _plain_rope(s):
    cos, sin = _angles(s["positions"], s["freqs"], s["axis"])
    x = s["input"].detach()
    y = _rotated(x, cos, sin, s["case"]["interleaved"]).to(x.dtype)
    if s["grad"] is None:
        return y
    return [y, _rotated(s["grad"], cos, -sin, s["case"]["interleaved"]).to(x.dtype)]


def _plain_linear(s):
    w, scales = s["weight"], s["scales"].float()
    n, k = w.shape[0], 2 * w.shape[1]
    codes = torch.stack((w & 15, w >> 4), -1).reshape(n, scales.shape[1], -1).float()
    zeros = 8.0 if s["zeros"] is None else s["zeros"].float()[..., None]
    y = s["input"].float() @ ((codes - zeros) * scales[..., None]).reshape(n, k).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["input"].dtype)


def _own_attention(s):
    return s["ops"].paged_attention(s["query"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"])


def _own_append(s):
    query = s["ops"].kv_append(s["key"], s["value"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"],
                               new_lengths=s["new_lengths"], query=s["query"], positions=s["positions"],
                               freqs=s["freqs"], sections=s["sections"], interleaved=s["case"]["interleaved"])
    return [s["k_cache"], s["v_cache"]] + ([] if query is None else [query])


def _own_rope(s):
    y = s["ops"].rope(s["input"], s["positions"], s["freqs"], sections=s["sections"],
                      interleaved=s["case"]["interleaved"])
    if s["grad"] is None:
        return y
    return [y.detach(), torch.autograd.grad(y, s["input"], s["grad"])[0]]


def _own_linear(s):
    return s["ops"].linear_w4(s["input"], s["weight"], s["scales"], s["zeros"], s["bias"])


_PLAIN = {"paged_attention": _plain_attention, "kv_append": _plain_append, "rope": _plain_rope,
          "linear_w4": _plain_linear}
_OWN = {"paged_attention": _own_attention, "kv_append": _own_append, "rope": _own_rope, "linear_w4": _own_linear}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# -------------------------------------------------------------------------------------------------
# what a pass cannot do without
# -------------------------------------------------------------------------------------------------

def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "paged_attention":
        total = sum(_lengths(case))
        rows = case["batch"] * case["heads"] * case["dim"]
        pages = sum(-(-n // case["page"]) for n in _lengths(case))
        return {"bytes": 2 * total * case["heads_kv"] * case["dim"] * size + 2 * rows * size + 4 * pages + 4 * case["batch"],
                "flops": 4 * total * case["heads"] * case["dim"]}
    if case["op"] == "kv_append":
        there = sum(_new_lengths(case))
        every = case["batch"] * case["tokens"]
        values = 4 * there * case["heads_kv"] * case["dim"] + 2 * every * case["heads"] * case["dim"]
        turned = there * (case["heads"] + case["heads_kv"]) * case["rot"]
        places = 0 if case["axes"] == 1 else 4 * case["axes"] * there
        return {"bytes": values * size + places + 8 * case["batch"], "flops": 3 * turned}
    if case["op"] == "rope":
        values = case["batch"] * case["heads"] * case["length"]
        ways = 2 if case["grad"] else 1
        return {"bytes": ways * 2 * values * case["dim"] * size + 4 * case["axes"] * case["batch"] * case["length"],
                "flops": ways * 3 * values * case["rot"]}
    m, n, k = case["tokens"], case["n"], case["k"]
    groups = n * (k // case["group"])
    return {"bytes": n * k // 2 + groups * (size + (1 if case["zeros"] else 0)) + (m * k + m * n) * size
            + (n * size if case["bias"] else 0), "flops": 2 * m * n * k}


# -------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# -------------------------------------------------------------------------------------------------

def _exact_turn(x, place, freqs, sections, interleaved, sign=1.0):
    """One [tokens, heads, dim] sequence turned, by complex products; place [axes, tokens]."""
    pairs = freqs.numel()
    out = x.double().clone()
    angle = torch.empty(x.shape[0], pairs, dtype=torch.float64, device=x.device)
    first = 0
    for axis, count in enumerate(sections or (pairs,)):
        angle[:, first:first + count] = torch.outer(place[axis].double(), freqs[first:first + count].double())
        first += count
    unit = torch.polar(torch.ones_like(angle), sign * angle)[:, None, :]
    j = torch.arange(pairs, device=x.device)
    real, imag = (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)
    z = torch.complex(out[..., real], out[..., imag]) * unit
    out[..., real], out[..., imag] = z.real, z.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "paged_attention":
        b, h, _, d = s["query"].shape
        out = torch.zeros(b, h, 1, d, dtype=torch.float64, device="cuda")
        group = h // case["heads_kv"]
        for i, n in enumerate(s["lengths"].tolist()):
            if n == 0:
                continue
            at = torch.arange(n, device="cuda")
            pages = s["page_table"][i].long()[at // case["page"]]
            for j in range(case["heads_kv"]):
                k, v = (s[c][pages, j, at % case["page"]].double() for c in ("k_cache", "v_cache"))
                q = s["query"][i, j * group:(j + 1) * group, 0].double()
                out[i, j * group:(j + 1) * group, 0] = torch.softmax(q @ k.t() * d ** -0.5, -1) @ v
        return out
    if case["op"] == "kv_append":
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        query = None if s["query"] is None else s["query"].double()
        total = s["lengths"].tolist()
        new = [case["tokens"]] * case["batch"] if s["new_lengths"] is None else s["new_lengths"].tolist()
        for i, (n, t) in enumerate(zip(total, new)):
            if t == 0:
                continue
            at = torch.arange(n - t, n, device="cuda")
            place = at[None] if s["positions"] is None else s["positions"][:, i, :t]
            pages = s["page_table"][i].long()[at // case["page"]]
            turn = (place, s["freqs"], s["sections"], case["interleaved"])
            k_cache[pages, :, at % case["page"]] = _exact_turn(s["key"][i, :, :t].transpose(0, 1), *turn)
            v_cache[pages, :, at % case["page"]] = s["value"][i, :, :t].transpose(0, 1).double()
            if query is not None:
                query[i, :, :t] = _exact_turn(s["query"][i, :, :t].transpose(0, 1), *turn).transpose(0, 1)
        return [k_cache, v_cache] + ([] if query is None else [query])
    if case["op"] == "rope":
        place = s["positions"][None] if s["sections"] is None else s["positions"]
        parts = [(s["input"].detach(), 1.0)] + ([] if s["grad"] is None else [(s["grad"], -1.0)])
        out = [torch.stack([_exact_turn(x[i].transpose(0, 1), place[:, i], s["freqs"], s["sections"],
                                        case["interleaved"], sign).transpose(0, 1) for i in range(x.shape[0])])
               for x, sign in parts]
        return out[0] if s["grad"] is None else out
    codes = torch.empty(case["n"], case["k"], dtype=torch.float64, device="cuda")
    codes[:, 0::2], codes[:, 1::2] = (s["weight"] % 16).double(), (s["weight"] // 16).double()
    out = torch.zeros(case["tokens"], case["n"], dtype=torch.float64, device="cuda")
    for g in range(case["k"] // case["group"]):
        cut = slice(g * case["group"], (g + 1) * case["group"])
        zero = 8.0 if s["zeros"] is None else s["zeros"][:, g:g + 1].double()
        out += (s["input"][:, cut].double() @ (codes[:, cut] - zero).t()) * s["scales"][:, g].double()
    return out if s["bias"] is None else out + s["bias"].double()
