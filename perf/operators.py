"""Measured cases of the attention operators: rotary positions, the 4-bit key/value cache and attention over it, attention over a prompt.

A case is a dict of plain values; lengths of ragged batches follow from its own numbers, so that ``work`` knows them.  With ``own``
false ``run`` computes an operator from elementary torch operations in 32 bits; with ``own`` true it makes the framework's calls.

Sequences are packed: a batch of B sequences is one tensor of all their tokens, sequence b in rows cu[b] .. cu[b + 1] - 1.  The cache
is paged: token t of sequence b lies in page block_table[b, t // page_size], at t % page_size; per head and token it holds head_dim
4-bit codes (element 2i in the low nibble), one fp16 scale and one 4-bit zero point for every block_size of them.
"""
import math
import os
import random
import sys

import torch

own = False

_TYPES = {"f16": torch.float16, "f32": torch.float32}
_context = None


def _framework():
    """The package, and this process's context."""
    global _context
    package = os.path.join(os.getcwd(), "onnx-vulkan-rs_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import ovk_b200
    if _context is None:
        _context = ovk_b200.Context(0)
    return ovk_b200, _context


def listed():
    return [
        # one decode step of a vision-language decoder (16 query and 2 key heads, time / height / width positions), 64 requests
        {"name": "rotary step", "op": "rotary", "dtype": "f16", "tokens": 64, "q_heads": 16, "kv_heads": 2, "head_dim": 128, "rotary_dim": 128,
         "axes": 3, "interleaved": False, "index": 64},
        # a packed prompt batch with images in it, same decoder
        {"name": "rotary prompt", "op": "rotary", "dtype": "f16", "tokens": 16411, "q_heads": 16, "kv_heads": 2, "head_dim": 128, "rotary_dim": 128,
         "axes": 3, "interleaved": False, "index": 64},
        # the new token of 64 requests goes into the cache
        {"name": "append step", "op": "append", "dtype": "f16", "batch": 64, "new": 1, "ragged": False, "context": 900, "kv_heads": 2, "head_dim": 128,
         "block_size": 32, "page_size": 16, "zero_points": True, "lens_seed": 1},
        # a batch of prompts goes into the cache; one wide key head, f32 activations
        {"name": "append prompt", "op": "append", "dtype": "f32", "batch": 24, "new": 900, "ragged": True, "context": 0, "kv_heads": 1, "head_dim": 256,
         "block_size": 64, "page_size": 64, "zero_points": True, "lens_seed": 2},
        # a dozen short chat prompts packed together
        {"name": "prompt short", "op": "prompt", "dtype": "f16", "batch": 12, "length": 90, "ragged": True, "before": 0, "q_heads": 16, "kv_heads": 2,
         "head_dim": 128, "causal": True, "window": 0, "lens_seed": 3},
        # one long document
        {"name": "prompt long", "op": "prompt", "dtype": "f16", "batch": 1, "length": 8192, "ragged": False, "before": 0, "q_heads": 16, "kv_heads": 2,
         "head_dim": 128, "causal": True, "window": 0, "lens_seed": 4},
        # the sliding-window layers of a decoder with 256-wide heads, three documents
        {"name": "prompt window", "op": "prompt", "dtype": "f16", "batch": 3, "length": 2500, "ragged": True, "before": 0, "q_heads": 4, "kv_heads": 1,
         "head_dim": 256, "causal": True, "window": 512, "lens_seed": 5},
        # an f32 graph: a chunk of new tokens after earlier ones, every query head with its own key head
        {"name": "prompt f32 chunk", "op": "prompt", "dtype": "f32", "batch": 4, "length": 600, "ragged": True, "before": 333, "q_heads": 8, "kv_heads": 8,
         "head_dim": 64, "causal": True, "window": 0, "lens_seed": 6},
        # one request in a chat, a decoder with one wide key head: latency
        {"name": "cache single", "op": "cache", "dtype": "f16", "batch": 1, "new": 1, "context": 900, "ragged": False, "q_heads": 4, "kv_heads": 1,
         "head_dim": 256, "window": 0, "block_size": 32, "page_size": 16, "zero_points": True, "lens_seed": 7},
        # a serving batch at ordinary contexts
        {"name": "cache batch", "op": "cache", "dtype": "f16", "batch": 48, "new": 1, "context": 4000, "ragged": True, "q_heads": 16, "kv_heads": 2,
         "head_dim": 128, "window": 0, "block_size": 32, "page_size": 16, "zero_points": True, "lens_seed": 8},
        # a few requests over very long contexts
        {"name": "cache long", "op": "cache", "dtype": "f16", "batch": 8, "new": 1, "context": 100000, "ragged": True, "q_heads": 16, "kv_heads": 2,
         "head_dim": 128, "window": 0, "block_size": 32, "page_size": 64, "zero_points": True, "lens_seed": 9},
        # four drafted tokens a request are verified at once, f32 graph, symmetric cache
        {"name": "cache drafts f32", "op": "cache", "dtype": "f32", "batch": 6, "new": 4, "context": 3000, "ragged": True, "q_heads": 8, "kv_heads": 4,
         "head_dim": 64, "window": 0, "block_size": 64, "page_size": 48, "zero_points": False, "lens_seed": 10},
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "prompt", "prompt", "cache", "cache"])
    dtype = rng.choice(["f16", "f16", "f32"])
    seed = rng.randrange(1 << 30)
    if op == "rotary":
        d = rng.choice([64, 80, 128, 256])
        heads = rng.choice([(4, 1), (16, 2), (8, 8), (7, 1), (32, 8)])
        return {"op": op, "dtype": dtype, "tokens": _between(rng, 1, 16384 * 18 * 128 // (d * sum(heads) * (2 if dtype == "f32" else 1))), "q_heads": heads[0],
                "kv_heads": heads[1], "head_dim": d, "rotary_dim": rng.choice([d, d, d // 2]), "axes": rng.choice([1, 2, 3]),
                "interleaved": rng.random() < 0.3, "index": rng.choice([32, 64])}
    if op == "append":
        d = rng.choice([64, 128, 256])
        hk = rng.choice([1, 2, 4, 8])
        batch = _between(rng, 1, 64)
        most = max(1, 5000000 // (batch * hk * d))
        return {"op": op, "dtype": dtype, "batch": batch, "new": _between(rng, 1, most), "ragged": rng.random() < 0.5, "context": rng.choice([0, _between(rng, 1, 2000)]),
                "kv_heads": hk, "head_dim": d, "block_size": rng.choice([b for b in (32, 64, 128) if d % b == 0]), "page_size": rng.choice([16, 64, 1, 50, 128]),
                "zero_points": rng.random() < 0.7, "lens_seed": seed}
    if op == "prompt":
        d = rng.choice([64, 80, 128, 256])
        hq, hk = rng.choice([(4, 1), (16, 2), (8, 8), (7, 1), (12, 4)])
        batch = _between(rng, 1, 16)
        most = int(math.sqrt((8192 * 8192 * 16 * 128 if dtype == "f16" else 2000 * 2000 * 8 * 128) / (7 * batch * hq * d)))
        return {"op": op, "dtype": dtype, "batch": batch, "length": _between(rng, 1, max(2, most)), "ragged": rng.random() < 0.7,
                "before": rng.choice([0, 0, _between(rng, 1, 500)]), "q_heads": hq, "kv_heads": hk, "head_dim": d, "causal": rng.random() < 0.75,
                "window": rng.choice([0, 0, _between(rng, 1, 1000)]), "lens_seed": seed}
    d = rng.choice([64, 128, 256])
    hq, hk = rng.choice([(4, 1), (16, 2), (8, 8), (7, 1), (12, 4)])
    batch = _between(rng, 1, 64)
    most = max(1, 8 * 100000 * 2 * 128 // (2 * batch * hk * d))
    return {"op": op, "dtype": dtype, "batch": batch, "new": rng.choice([1, 1, 1, 2, 5]), "context": _between(rng, 1, min(most, 131072)), "ragged": rng.random() < 0.7,
            "q_heads": hq, "kv_heads": hk, "head_dim": d, "window": rng.choice([0, 0, 0, 512]),
            "block_size": rng.choice([b for b in (32, 64, 128) if d % b == 0]), "page_size": rng.choice([16, 64, 48, 100]), "zero_points": rng.random() < 0.7,
            "lens_seed": seed}


def _lengths(case, mean):
    """Lengths of the batch's sequences: the mean, or from a quarter of it to about twice it."""
    if not case["ragged"]:
        return [mean] * case["batch"]
    r = random.Random(case["lens_seed"])
    return [max(1, int(mean * r.uniform(0.25, 1.75))) for _ in range(case["batch"])]


def _starts(lengths, device):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=device)


def _pairs(new, total, causal, window):
    """How many (query, key) pairs the queries at the end of a sequence of `total` tokens attend."""
    n = 0
    for i in range(new):
        last = total - new + i if causal else total - 1
        first = max(0, total - new + i - window + 1) if window else 0
        n += max(0, last - first + 1)
    return n


def _sections(case):
    pairs = case["rotary_dim"] // 2
    if case["axes"] == 1:
        return [pairs]
    first = pairs // 4
    if case["axes"] == 2:
        return [first, pairs - first]
    rest = pairs - first
    return [first, rest // 2, rest - rest // 2]


def work(case):
    size = 2 if case["dtype"] == "f16" else 4
    d = case["head_dim"]
    if case["op"] == "rotary":
        n = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        rows = min(case["tokens"], 8192)  # a position's row of the tables is read from memory once
        return {"bytes": 2 * n * d * size + rows * case["rotary_dim"] * 4 + case["tokens"] * case["axes"] * case["index"] // 8,
                "flops": 3 * n * case["rotary_dim"]}
    hk = case["kv_heads"]
    if case["op"] in ("append", "cache"):
        blocks = d // case["block_size"]
        row = d // 2 + 2 * blocks + ((blocks + 1) // 2 if case["zero_points"] else 0)
    if case["op"] == "append":  # the rows in, their codes, and the values that the codes stand for
        n = sum(_lengths(case, case["new"])) * hk * 2
        return {"bytes": n * (2 * d * size + row), "flops": 6 * n * d}
    if case["op"] == "prompt":
        new = _lengths(case, case["length"])
        pairs = sum(_pairs(n, n + case["before"], case["causal"], case["window"]) for n in new)
        q, k = sum(new), sum(n + case["before"] for n in new)
        return {"bytes": 2 * d * size * (q * case["q_heads"] + k * hk), "flops": 4 * d * case["q_heads"] * pairs}
    new = case["new"]
    pairs = seen = 0
    for n in _lengths(case, case["context"]):
        pairs += _pairs(new, n, True, case["window"])
        seen += min(n, case["window"] + new - 1) if case["window"] else n
    return {"bytes": seen * hk * 2 * row + 2 * case["batch"] * new * case["q_heads"] * d * size, "flops": 4 * d * case["q_heads"] * pairs}


def _rows(shape, generator, spread):
    """Activations with the outlier channels that keys and values have."""
    x = torch.randn(shape, generator=generator, device="cuda")
    return x * spread


def _spread(heads, d, generator):
    s = 0.5 + torch.rand((heads, d), generator=generator, device="cuda")
    return torch.where(torch.rand((heads, d), generator=generator, device="cuda") < 0.02, 3 * s, s)


def _quantize(x, block, zero_points):
    """Codes, scales and zero points (4-bit values, or None) of the blocks along the last axis; in 64 bits, since a quotient next to a
    border must go to the same code everywhere."""
    x = x.double().reshape(*x.shape[:-1], x.shape[-1] // block, block)
    lo, hi = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
    of = lambda v: torch.full((), v, dtype=torch.float64, device=x.device)  # noqa: E731 - a tensor, so that the division is one
    if zero_points:
        scale = ((hi - lo) / of(15.0)).clamp(max=65504).half()
    else:
        scale = torch.maximum(hi / of(7.0), -lo / of(8.0)).clamp(max=65504).half()
    s = scale.double()
    safe = torch.where(s > 0, s, torch.ones_like(s))
    if zero_points:
        zero = torch.where(s > 0, torch.round(-lo / safe).clamp(0, 15), torch.zeros_like(s))
    else:
        zero = torch.full_like(s, 8)
    code = (torch.where(s[..., None] > 0, torch.round(x / safe[..., None]), torch.zeros_like(x)) + zero[..., None]).clamp(0, 15)
    return code.flatten(-2).to(torch.uint8), scale, zero.to(torch.uint8)


def _pack(v):
    """Two 4-bit values a byte along the last axis, the first in the low nibble."""
    if v.shape[-1] % 2:
        v = torch.nn.functional.pad(v, (0, 1))
    return v[..., 0::2] | (v[..., 1::2] << 4)


def _unpack(v, n):
    return torch.stack((v & 15, v >> 4), -1).flatten(-2)[..., :n]


def _cache(case, pages, generator, empty):
    hk, d, ps, block = case["kv_heads"], case["head_dim"], case["page_size"], case["block_size"]
    made = {}
    for name in ("k", "v"):
        if empty:
            code = torch.zeros((pages, hk, ps, d), dtype=torch.uint8, device="cuda")
            scale = torch.zeros((pages, hk, ps, d // block), dtype=torch.float16, device="cuda")
            zero = torch.zeros((pages, hk, ps, d // block), dtype=torch.uint8, device="cuda")
        else:
            x = _rows((pages, hk, ps, d), generator, _spread(hk, d, generator)[:, None, :])
            code, scale, zero = _quantize(x, block, case["zero_points"])
            del x
        made[name] = _pack(code)
        made[name + "_scales"] = scale
        made[name + "_zero_points"] = _pack(zero) if case["zero_points"] else None
    return made


def _paged(case, totals, generator):
    """A block table whose pages lie anywhere, and how many pages there are."""
    per = [-(-n // case["page_size"]) for n in totals]
    pages = sum(per) + 3
    order = torch.randperm(pages, generator=generator, device="cuda").int()
    table = torch.zeros((len(totals), max(max(per), 1)), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def _handle(state):
    """The framework's description of the cache, made once as a program does."""
    if own:
        ovk, _ = _framework()
        state["handle"] = ovk.KV4Cache(**state["cache"])
    return state


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t, d, hk = _TYPES[case["dtype"]], case["head_dim"], case["kv_heads"]
    if case["op"] == "rotary":
        n, pairs, far = case["tokens"], case["rotary_dim"] // 2, 8192
        angle = torch.arange(far, device="cuda").double()[:, None] * torch.pow(torch.tensor(1e6, device="cuda", dtype=torch.float64),
                                                                              -torch.arange(pairs, device="cuda").double() / pairs)
        # text counts along every axis alike; images spread height and width over a grid
        at = torch.arange(n, device="cuda") % far
        image = torch.rand((n,), generator=g, device="cuda") < 0.5
        positions = torch.stack([at] + [torch.where(image, torch.randint(0, far, (n,), generator=g, device="cuda"), at) for _ in range(case["axes"] - 1)])
        return {"case": case, "q": _rows((n, case["q_heads"], d), g, 1.0).to(t), "k": _rows((n, hk, d), g, _spread(hk, d, g)).to(t),
                "cos": angle.cos().float(), "sin": angle.sin().float(), "positions": positions.to(torch.int64 if case["index"] == 64 else torch.int32).contiguous(),
                "sections": _sections(case)}
    if case["op"] == "append":
        new = _lengths(case, case["new"])
        totals = [n + case["context"] for n in new]
        table, pages = _paged(case, totals, g)
        cu, lens = _starts(new, "cuda"), torch.tensor(totals, dtype=torch.int32, device="cuda")
        token = torch.arange(sum(new), device="cuda")
        b = torch.searchsorted(cu[1:].long(), token, right=True)
        at = lens[b].long() - (cu[b + 1].long() - token)
        row = (table[b, at // case["page_size"]].long()[:, None] * hk + torch.arange(hk, device="cuda")) * case["page_size"] + (at % case["page_size"])[:, None]
        return _handle({"case": case, "k": _rows((sum(new), hk, d), g, _spread(hk, d, g)).to(t), "v": _rows((sum(new), hk, d), g, _spread(hk, d, g)).to(t),
                        "cache": _cache(case, pages, g, True), "table": table, "cu": cu, "lens": lens, "rows": row})
    if case["op"] == "prompt":
        new = _lengths(case, case["length"])
        seen = [n + case["before"] for n in new]
        cu_q, cu_k = _starts(new, "cuda"), _starts(seen, "cuda")
        return {"case": case, "q": _rows((sum(new), case["q_heads"], d), g, 1.3).to(t), "k": _rows((sum(seen), hk, d), g, _spread(hk, d, g)).to(t),
                "v": _rows((sum(seen), hk, d), g, _spread(hk, d, g)).to(t), "cu_q": cu_q, "cu_k": cu_k if case["before"] else cu_q, "longest": max(new),
                "furthest": max(seen), "scale": 1 / math.sqrt(d)}
    totals = _lengths(case, case["context"])
    table, pages = _paged(case, totals, g)
    n = case["batch"] * case["new"]
    return _handle({"case": case, "q": _rows((n, case["q_heads"], d), g, 1.3).to(t), "cache": _cache(case, pages, g, False), "table": table,
                    "cu": _starts([case["new"]] * case["batch"], "cuda"), "lens": torch.tensor(totals, dtype=torch.int32, device="cuda"), "furthest": max(totals),
                    "scale": 1 / math.sqrt(d)})


# ------------------------------------------------------------------ plain forms
def _rotated(x, cos, sin, case):
    """cos, sin: [tokens, pairs], in 32 bits."""
    r, c, s = case["rotary_dim"], cos[:, None], sin[:, None]
    y = x.float()
    if case["interleaved"]:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = y[..., :r // 2], y[..., r // 2:r]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turned, y[..., r:]), -1).to(x.dtype)


def _plain_rotary(s):
    case = s["case"]
    axis = torch.repeat_interleave(torch.arange(case["axes"], device="cuda"), torch.tensor(s["sections"], device="cuda"))
    at = s["positions"].long()[axis].t()  # [tokens, pairs]
    column = torch.arange(at.shape[1], device="cuda")
    cos, sin = s["cos"][at, column], s["sin"][at, column]
    return _rotated(s["q"], cos, sin, case), _rotated(s["k"], cos, sin, case)


def _plain_append(s):
    case, cache, out = s["case"], s["cache"], []
    block, ps, cu = case["block_size"], case["page_size"], s["cu"].long()
    token = torch.arange(s["k"].shape[0], device="cuda")
    b = torch.searchsorted(cu[1:], token, right=True)
    at = s["lens"].long()[b] - (cu[b + 1] - token)
    page, off = s["table"][b, at // ps].long(), at % ps
    for name in ("k", "v"):
        code, scale, zero = _quantize(s[name], block, case["zero_points"])
        cache[name][page, :, off] = _pack(code)
        cache[name + "_scales"][page, :, off] = scale
        if case["zero_points"]:
            cache[name + "_zero_points"][page, :, off] = _pack(zero)
        out.append(_values(cache, name, s["rows"], case).to(s[name].dtype))
    return tuple(out)


def _values(cache, name, rows, case):
    """f32 values of cache rows given by their index over pages, heads and places."""
    d, blocks = case["head_dim"], case["head_dim"] // case["block_size"]
    code = _unpack(cache[name].flatten(0, 2)[rows], d).float().unflatten(-1, (blocks, case["block_size"]))
    scale = cache[name + "_scales"].flatten(0, 2)[rows].float()
    zero = _unpack(cache[name + "_zero_points"].flatten(0, 2)[rows], blocks).float() if case["zero_points"] else torch.full_like(scale, 8)
    return ((code - zero[..., None]) * scale[..., None]).flatten(-2)


def _attend(q, k, v, keep, scale):
    """q [B, Hk, G, N, D], k and v [B, Hk, L, D], keep [B, N, L]: softmax attention in 32 bits; a row that attends nothing is zero."""
    score = torch.matmul(q, k[:, :, None].transpose(-1, -2)) * scale
    score = score.masked_fill(~keep[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v[:, :, None]) / torch.where(total > 0, total, torch.ones_like(total))


def _keep(new, seen, longest, furthest, causal, window):
    """[B, longest, furthest]: which keys the queries at the end of each sequence attend."""
    i = torch.arange(longest, device="cuda")[None, :, None]
    j = torch.arange(furthest, device="cuda")[None, None]
    at = i + (seen - new)[:, None, None]
    keep = (j < seen[:, None, None]) & (i < new[:, None, None])
    if causal:
        keep = keep & (j <= at)
    if window:
        keep = keep & (j > at - window)
    return keep


def _padded(x, cu, longest):
    """[B, longest, ...] of a packed tensor; rows past a sequence's end repeat some row and are masked later."""
    at = cu[:-1].long()[:, None] + torch.arange(longest, device="cuda")
    return x[at.clamp(max=x.shape[0] - 1)]


def _packed(x, cu, tokens):
    token = torch.arange(tokens, device="cuda")
    b = torch.searchsorted(cu[1:].long(), token, right=True)
    return x[b, token - cu.long()[b]]


def _plain_prompt(s):
    case = s["case"]
    hq, hk = case["q_heads"], case["kv_heads"]
    new, seen = (s[c].long()[1:] - s[c].long()[:-1] for c in ("cu_q", "cu_k"))
    q = _padded(s["q"], s["cu_q"], s["longest"]).float().unflatten(2, (hk, hq // hk)).permute(0, 2, 3, 1, 4)
    k, v = (_padded(s[c], s["cu_k"], s["furthest"]).float().transpose(1, 2) for c in ("k", "v"))
    o = _attend(q, k, v, _keep(new, seen, s["longest"], s["furthest"], case["causal"], case["window"]), s["scale"])
    return _packed(o.permute(0, 3, 1, 2, 4).flatten(2, 3), s["cu_q"], s["q"].shape[0]).to(s["q"].dtype)


def _plain_cache(s):
    case, far = s["case"], s["furthest"]
    hq, hk, ps = case["q_heads"], case["kv_heads"], case["page_size"]
    at = torch.arange(far, device="cuda")
    rows = (s["table"][:, at // ps].long()[:, None] * hk + torch.arange(hk, device="cuda")[None, :, None]) * ps + at % ps  # [B, Hk, L]
    k, v = _values(s["cache"], "k", rows, case), _values(s["cache"], "v", rows, case)
    q = s["q"].float().unflatten(0, (case["batch"], case["new"])).unflatten(2, (hk, hq // hk)).permute(0, 2, 3, 1, 4)
    new = torch.full_like(s["lens"], case["new"]).long()
    o = _attend(q, k, v, _keep(new, s["lens"].long(), case["new"], far, True, case["window"]), s["scale"])
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3).flatten(0, 1).to(s["q"].dtype)


def run(state):
    s, case = state, state["case"]
    if own:
        _, ctx = _framework()
        if case["op"] == "rotary":
            return ctx.rotary(s["q"], s["cos"], s["sin"], s["positions"], k=s["k"], sections=s["sections"], interleaved=case["interleaved"])
        if case["op"] == "append":
            cache = s["handle"]
            ctx.kv4_append(cache, s["k"], s["v"], s["table"], s["cu"], s["lens"])
            k = ctx.gather_block_quantized(cache.k.flatten(0, 2), s["rows"], cache.k_scales, cache.k_zero_points, case["block_size"], out_dtype=s["k"].dtype)
            v = ctx.gather_block_quantized(cache.v.flatten(0, 2), s["rows"], cache.v_scales, cache.v_zero_points, case["block_size"], out_dtype=s["v"].dtype)
            return k, v
        if case["op"] == "prompt":
            return ctx.attention_prompt(s["q"], s["k"], s["v"], s["cu_q"], s["longest"], cu_k=s["cu_k"], scale=s["scale"], causal=case["causal"],
                                        window=case["window"])
        return ctx.attention_kv4(s["handle"], s["q"], s["table"], s["cu"], s["lens"], max_tokens=case["new"], scale=s["scale"], window=case["window"])
    return {"rotary": _plain_rotary, "append": _plain_append, "prompt": _plain_prompt, "cache": _plain_cache}[case["op"]](s)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    """From the definitions, one sequence and one key head at a time."""
    cost = work(case)["flops"]
    if cost > 4e12:
        return None
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return tuple(_exact_rotary(s[c].double(), s, case) for c in ("q", "k"))
    if case["op"] == "append":
        return tuple(_exact_rounded(s[c].double(), case) for c in ("k", "v"))
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros((s["q"].shape[0], hq, d), dtype=torch.float64, device="cuda")
    if case["op"] == "prompt":
        cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
        spans = [(cu_q[b], cu_q[b + 1], cu_k[b + 1] - cu_k[b]) for b in range(case["batch"])]
        causal = case["causal"]
    else:
        lens = s["lens"].tolist()
        spans = [(b * case["new"], (b + 1) * case["new"], lens[b]) for b in range(case["batch"])]
        causal = True
    for b, (first, end, total) in enumerate(spans):
        key = torch.arange(total, device="cuda")
        for h in range(hk):
            if case["op"] == "prompt":
                k, v = (s[c][cu_k[b]:cu_k[b + 1], h].double() for c in ("k", "v"))
            else:
                page = s["table"][b].long()[key // case["page_size"]]
                k, v = (_exact_values(s["cache"], c, page, h, key % case["page_size"], case) for c in ("k", "v"))
            group = slice(h * (hq // hk), (h + 1) * (hq // hk))
            for lo in range(first, end, 1024):
                hi = min(end, lo + 1024)
                place = total - (end - torch.arange(lo, hi, device="cuda"))[:, None]
                allowed = torch.ones((hi - lo, total), dtype=torch.bool, device="cuda")
                if causal:
                    allowed &= key <= place
                if case["window"]:
                    allowed &= key > place - case["window"]
                logit = torch.einsum("ngd,ld->gnl", s["q"][lo:hi, group].double(), k) * s["scale"]
                weight = torch.softmax(torch.where(allowed, logit, torch.full_like(logit, -1e300)), -1) * allowed
                out[lo:hi, group] = torch.einsum("gnl,ld->ngd", weight, v)
    return out


def _exact_rotary(x, s, case):
    out, r = x.clone(), case["rotary_dim"]
    begin = 0
    for axis, count in enumerate(s["sections"]):
        pair = torch.arange(begin, begin + count, device="cuda")
        row = s["positions"][axis].long()[:, None]
        c, n = s["cos"].double()[row, pair][:, None], s["sin"].double()[row, pair][:, None]
        i, j = (2 * pair, 2 * pair + 1) if case["interleaved"] else (pair, pair + r // 2)
        out[..., i] = x[..., i] * c - x[..., j] * n
        out[..., j] = x[..., j] * c + x[..., i] * n
        begin += count
    return out


def _exact_rounded(x, case):
    """What the cache holds of x: each block in sixteen steps of an fp16 scale."""
    b = x.unflatten(-1, (-1, case["block_size"]))
    low, high = b.amin(-1, keepdim=True).clamp(max=0), b.amax(-1, keepdim=True).clamp(min=0)
    step = ((high - low) / 15 if case["zero_points"] else torch.maximum(high / 7, -low / 8)).half().double()
    zero = torch.round(-low / step).clamp(0, 15) if case["zero_points"] else torch.full_like(step, 8)
    return (((torch.round(b / step) + zero).clamp(0, 15) - zero) * step).flatten(-2)


def _exact_values(cache, name, page, head, place, case):
    d, block = case["head_dim"], case["block_size"]
    element = torch.arange(d, device="cuda")
    byte = cache[name][page, head, place].long()
    code = (byte[:, element // 2] >> (4 * (element % 2))) & 15
    which = element // block
    scale = cache[name + "_scales"][page, head, place].double()[:, which]
    if case["zero_points"]:
        zero = (cache[name + "_zero_points"][page, head, place].long()[:, which // 2] >> (4 * (which % 2))) & 15
    else:
        zero = torch.full_like(code, 8)
    return (code - zero).double() * scale
