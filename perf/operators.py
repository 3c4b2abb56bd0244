"""The operators of an 8-bit decoder layer as cases to time: what a program that serves a language model calls per layer.

  quantize  the activations of a layer, one scale per token (``serving.quantize_rows``)
  linear    a projection: activations quantised per token, times int8 weights with a scale per channel
            (``serving.QuantizedLinear``)
  append    new keys and values, rotated by their positions, into a paged int8 cache with a scale per page and head; the
            queries are rotated in the same call (``serving.PagedCache.append``)
  attend    attention of the new tokens over that cache (``serving.PagedCache.attend``)

``run`` computes a case in its plain form (elementary torch operations in 32 bits; in 64 what decides between two whole
numbers), or, where ``own`` is true, by the calls that a user makes of the framework.  ``exact`` computes it from the
operator's definition in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # a decode step's activations in front of a projection: a few hundred kilobytes, launch-bound
        {"name": "quantize_24x5120", "op": "quantize", "m": 24, "k": 5120, "dtype": "bf16"},
        # a whole prompt batch's activations
        {"name": "quantize_8192x8192", "op": "quantize", "m": 8192, "k": 8192, "dtype": "f16"},
        # one token of one conversation: the weights' bytes are all there is
        {"name": "linear_1x4096x4096", "op": "linear", "m": 1, "k": 4096, "n": 4096, "dtype": "bf16", "bias": False},
        # a decode batch through a wide projection
        {"name": "linear_56x8192x10240", "op": "linear", "m": 56, "k": 8192, "n": 10240, "dtype": "f16", "bias": True},
        # a pruned layer: no size is a multiple of anything
        {"name": "linear_1003x2565x1390", "op": "linear", "m": 1003, "k": 2565, "n": 1390, "dtype": "f32", "bias": True},
        # a prompt batch: the tensor cores' case
        {"name": "linear_8192x8192x8192", "op": "linear", "m": 8192, "k": 8192, "n": 8192, "dtype": "bf16", "bias": False},
        # a decode step of 64 conversations, small pages
        {"name": "append_64x1", "op": "append", "b": 64, "new": 1, "prior": 40, "hq": 32, "hkv": 8, "d": 128, "rot": 128,
         "page": 16, "interleaved": False, "dtype": "bf16", "mix": 1},
        # prompts of a few conversations, some of them continued; part of each head rotated, in neighbouring pairs
        {"name": "append_6x1800", "op": "append", "b": 6, "new": 1800, "prior": 200, "hq": 32, "hkv": 8, "d": 128, "rot": 64,
         "page": 64, "interleaved": True, "dtype": "f16", "mix": 2},
        # a decode step of a few short conversations
        {"name": "attend_8x1_700", "op": "attend", "b": 8, "new": 1, "prior": 700, "hq": 32, "hkv": 8, "d": 128, "page": 16,
         "window": 0, "cap": 0.0, "dtype": "bf16", "mix": 3},
        # a decode step over long conversations: some 650 MB of cache
        {"name": "attend_32x1_16000", "op": "attend", "b": 32, "new": 1, "prior": 16000, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "window": 0, "cap": 0.0, "dtype": "bf16", "mix": 4},
        # chunks of prompts through a layer with a sliding window and capped scores, wide heads
        {"name": "attend_3x300_4500", "op": "attend", "b": 3, "new": 300, "prior": 4500, "hq": 16, "hkv": 8, "d": 256,
         "page": 32, "window": 1024, "cap": 50.0, "dtype": "f16", "mix": 5},
        # whole prompts
        {"name": "attend_4x6000", "op": "attend", "b": 4, "new": 6000, "prior": 0, "hq": 32, "hkv": 8, "d": 128, "page": 64,
         "window": 0, "cap": 0.0, "dtype": "bf16", "mix": 6},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _width(rng, lo, hi):
    """A feature count: mostly a multiple of 64 or 16, otherwise any number."""
    k = _log(rng, lo, hi)
    r = rng.random()
    step = 64 if r < 0.5 else 16 if r < 0.75 else 1
    return max(lo, k // step * step)


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "append", "attend", "attend"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "quantize":
        return {"op": op, "m": _log(rng, 1, 8192), "k": _width(rng, 64, 8192), "dtype": rng.choice(["bf16", "f16", "f32"])}
    if op == "linear":
        return {"op": op, "m": _log(rng, 1, 8000), "k": _width(rng, 64, 8192), "n": _width(rng, 64, 8192),
                "dtype": rng.choice(["bf16", "f16", "f32"]), "bias": rng.random() < 0.5}
    d = rng.choice([64, 64, 128, 128, 128, 256, 80, 96])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 4, 5, 8])
    c = {"op": op, "hq": hq, "hkv": hkv, "d": d, "page": rng.choice([16, 16, 32, 48, 64, 128]), "dtype": dtype,
         "mix": rng.randrange(1 << 20)}
    if op == "append":
        c["b"] = _log(rng, 1, 96)
        c["new"] = rng.choice([1, 1, 1, _log(rng, 2, 8)]) if rng.random() < 0.6 else _log(rng, 2, max(2, 8000 // c["b"]))
        c["prior"] = rng.choice([0, _log(rng, 1, 300)])
        c["rot"] = rng.choice([d, d, d // 2])
        c["interleaved"] = rng.random() < 0.4
        return c
    c["window"] = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
    c["cap"] = rng.choice([0.0, 0.0, 0.0, 30.0])
    kind = rng.random()
    if kind < 0.5:  # single tokens, or a few that a draft model proposed
        c["b"] = _log(rng, 1, 64)
        c["new"] = rng.choice([1, 1, 1, _log(rng, 2, 8)])
        c["prior"] = _log(rng, 1, 250000 // c["b"])
    elif kind < 0.75:  # chunks
        c["b"] = _log(rng, 1, 6)
        c["new"] = _log(rng, 16, 512)
        c["prior"] = _log(rng, 1, 10000)
    else:  # prompts
        c["b"] = _log(rng, 1, 8)
        c["new"] = _log(rng, 64, 20000 // c["b"])
        c["prior"] = 0
    while work(c)["flops"] > 5e11:  # no more than the longest listed prompts
        c["new"] = max(1, c["new"] // 2)
    return c


def _ragged(c):
    """New and older tokens of each sequence: the first has the most of both, the others anything from a quarter of it on."""
    r = random.Random(c["mix"])
    new, prior = [c["new"]], [c["prior"]]
    for _ in range(c["b"] - 1):
        new.append(max(1, int(c["new"] * r.uniform(0.25, 1.0))))
        prior.append(int(c["prior"] * r.uniform(0.25, 1.0)))
    return new, prior


def _attended(n, old, window):
    """Pairs of query and key, and keys that any of the n queries sees, of one sequence with `old` earlier tokens."""
    total = old + n
    if window <= 0:
        return n * old + n * (n + 1) // 2, total
    pairs = sum(min(old + i + 1, window) for i in range(n))
    return pairs, min(total, window + n - 1)


def work(case):
    op = case["op"]
    if op == "quantize":
        m, k = case["m"], case["k"]
        # the values come back as 32-bit floats
        return {"bytes": m * k * (_TYPES[case["dtype"]].itemsize + 4) + 4 * m, "flops": 2 * m * k}
    if op == "linear":
        m, k, n, t = case["m"], case["k"], case["n"], _TYPES[case["dtype"]].itemsize
        return {"bytes": m * k * t + n * k + 4 * n * (2 if case["bias"] else 1) + m * n * t, "flops": 2 * m * k * n}
    new, prior = _ragged(case)
    tokens, d, hq, hkv, t = sum(new), case["d"], case["hq"], case["hkv"], _TYPES[case["dtype"]].itemsize
    if op == "append":
        cache = _pool(case) * hkv * case["page"] * d
        # the cache's values come back as 32-bit floats
        return {"bytes": tokens * d * t * (2 * hkv + 2 * hq) + 8 * cache + 4 * tokens * case["rot"],
                "flops": 6 * tokens * d * (hq + 2 * hkv)}
    pairs, keys = 0, 0
    for n, old in zip(new, prior):
        p, k = _attended(n, old, case["window"])
        pairs, keys = pairs + p, keys + k
    return {"bytes": 2 * tokens * hq * d * t + 2 * keys * hkv * d, "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------- inputs

def _pool(case):
    new, prior = _ragged(case)
    pages = sum((n + old + case["page"] - 1) // case["page"] for n, old in zip(new, prior))
    return pages + 3


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    dev = "cuda"
    if case["op"] in ("quantize", "linear"):
        dtype, m, k = _TYPES[case["dtype"]], case["m"], case["k"]
        x = torch.randn(m, k, generator=g, device=dev)
        # a few features carry large values, as the residual stream of a trained model does
        loud = torch.rand(k, generator=g, device=dev) < 0.002
        s["x"] = torch.where(loud, 12 * x, x).to(dtype)
        if case["op"] == "linear":
            n = case["n"]
            s["w"] = (torch.randn(n, k, generator=g, device=dev) * 32).round_().clamp_(-127, 127).to(torch.int8)
            s["ws"] = (0.5 + torch.rand(n, generator=g, device=dev)) * (k ** -0.5 / 32)
            s["bias"] = torch.randn(n, generator=g, device=dev) * 0.1 if case["bias"] else None
            if own:
                s["linear"] = _serving().QuantizedLinear(s["w"], s["ws"], s["bias"])
        return s
    dtype, d, hq, hkv, page = _TYPES[case["dtype"]], case["d"], case["hq"], case["hkv"], case["page"]
    new, prior = _ragged(case)
    tokens, pool = sum(new), _pool(case)
    s["new"], s["prior"] = new, prior
    s["starts"] = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device=dev)
    s["lengths"] = torch.tensor([n + old for n, old in zip(new, prior)], dtype=torch.int32, device=dev)
    s["max_new"], s["max_length"] = max(new), max(n + old for n, old in zip(new, prior))
    width = (s["max_length"] + page - 1) // page
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(new), width, dtype=torch.int32, device=dev)
    at = 0
    for i, (n, old) in enumerate(zip(new, prior)):
        count = (n + old + page - 1) // page
        table[i, :count] = order[at:at + count]
        at += count
    s["table"] = table
    # cache[0]: keys, cache[1]: values
    cache = torch.empty(2, pool, hkv, page, d, dtype=torch.int8, device=dev)
    for part in cache.view(2 * pool, -1).split(4096):
        part.copy_(torch.randn(part.shape, generator=g, device=dev).mul_(36).round_().clamp_(-127, 127))
    scales = (0.6 + 0.8 * torch.rand(2, pool, hkv, generator=g, device=dev)) / 36
    s["cache"], s["scales"] = cache, scales
    s["q"] = (1.5 * torch.randn(tokens, hq, d, generator=g, device=dev)).to(dtype)
    if case["op"] == "append":
        s["k"] = torch.randn(tokens, hkv, d, generator=g, device=dev).to(dtype)
        s["v"] = torch.randn(tokens, hkv, d, generator=g, device=dev).to(dtype)
        half = case["rot"] // 2
        angle = torch.arange(s["max_length"], dtype=torch.float64, device=dev)[:, None] * (
            10000.0 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half))
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    if own:
        s["paged"] = _serving().PagedCache(cache, scales)
        s["batch"] = _serving().PagedBatch(s["starts"], s["lengths"], table, s["max_new"], s["max_length"])
    return s


def _serving():
    from __graft_entry__ import load_package
    load_package()
    from mlel_b200 import serving
    return serving


# ---------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    return (_RUN_OWN if own else _RUN_PLAIN)[op](state)


def _own_quantize(s):
    q, scales = _serving().quantize_rows(s["x"])
    return q * scales[:, None], scales


def _own_linear(s):
    return s["linear"](s["x"])


def _own_append(s):
    q = s["paged"].append(s["k"], s["v"], s["cos"], s["sin"], s["batch"], q=s["q"], interleaved=s["case"]["interleaved"])
    return q, s["cache"] * s["scales"][..., None, None]


def _own_attend(s):
    return s["paged"].attend(s["q"], s["batch"], window=s["case"]["window"], softcap=s["case"]["cap"])


def _plain_rows(x):
    """Rows in 8 bits: whole numbers as floats, and a scale per row."""
    scales = (x.abs().amax(dim=1).double() / 127).float()
    q = torch.round(x.double() / scales.double()[:, None]).clamp(-127, 127).float()
    return torch.where(scales[:, None] > 0, q, torch.zeros_like(q)), scales


def _plain_quantize(s):
    q, scales = _plain_rows(s["x"])
    return q * scales[:, None], scales


def _plain_linear(s):
    q, scales = _plain_rows(s["x"])
    y = (q @ s["w"].float().t()) * scales[:, None] * s["ws"][None, :]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _plain_rotate(x, cos, sin, rot, interleaved):
    """x [tokens, heads, d] in 32 or 64 bits, cos and sin [tokens, rot / 2]."""
    cos, sin = cos.to(x.dtype)[:, None, :], sin.to(x.dtype)[:, None, :]
    turned, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _plain_append(s):
    c = s["case"]
    page, rot = c["page"], c["rot"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    tokens = s["q"].shape[0]
    index = torch.arange(tokens, device=starts.device)
    seq = torch.searchsorted(starts[1:], index, right=True)
    position = lengths[seq] - starts[seq + 1] + index
    slot, offset = s["table"][seq, position // page].long(), position % page
    cos, sin = s["cos"][position], s["sin"][position]
    q = _plain_rotate(s["q"].float(), cos, sin, rot, c["interleaved"]).to(s["q"].dtype)
    k = _plain_rotate(s["k"].double(), cos, sin, rot, c["interleaved"])
    pool = s["cache"].shape[1]
    first = torch.full((pool,), page, dtype=torch.int64, device=starts.device)
    first.scatter_reduce_(0, slot, offset, "amin")  # tokens that a page held before; `page` where nothing is new
    for side, x in enumerate((k, s["v"].double())):
        cache, scales = s["cache"][side], s["scales"][side]
        most = torch.zeros_like(scales, dtype=x.dtype).index_reduce_(0, slot, x.abs().amax(dim=-1), "amax")
        old = torch.where(first[:, None] > 0, scales, torch.zeros_like(scales))
        now = torch.maximum(old, (most / 127).float())
        grown = (now > old) & (old > 0)
        older = torch.arange(page, device=starts.device)[None, :] < first[:, None]
        by = torch.where(grown, now, torch.ones_like(now)).double()[..., None, None]
        again = torch.round(cache.double() * old.double()[..., None, None] / by).to(torch.int8)
        cache.copy_(torch.where(older[:, None, :, None] & grown[..., None, None], again, cache))
        scales.copy_(torch.where(first[:, None] < page, now, scales))
        by = now[slot].double()[..., None]
        numbers = torch.where(by > 0, torch.round(x / by).clamp(-127, 127), torch.zeros_like(x))
        cache[slot, :, offset] = numbers.to(torch.int8)
    return q, s["cache"] * s["scales"][..., None, None]


def _plain_attend(s):
    c = s["case"]
    hq, hkv, d, page, window, cap = c["hq"], c["hkv"], c["d"], c["page"], c["window"], c["cap"]
    group, scale = hq // hkv, d ** -0.5
    out = torch.empty_like(s["q"])
    at = 0
    for i, (n, old) in enumerate(zip(s["new"], s["prior"])):
        total = n + old
        pages = s["table"][i, :(total + page - 1) // page].long()
        key_at = torch.arange(total, device=pages.device)[None, :]
        query_at = old + torch.arange(n, device=pages.device)[:, None]
        seen = key_at <= query_at
        if window > 0:
            seen &= key_at > query_at - window
        for h in range(hkv):
            k = (s["cache"][0, pages, h].float() * s["scales"][0, pages, h][:, None, None]).reshape(-1, d)[:total]
            v = (s["cache"][1, pages, h].float() * s["scales"][1, pages, h][:, None, None]).reshape(-1, d)[:total]
            q = s["q"][at:at + n, h * group:(h + 1) * group].float().transpose(0, 1)
            score = (q @ k.t()) * scale
            if cap > 0:
                score = torch.tanh(score / cap) * cap
            score = score.masked_fill(~seen, -math.inf)
            top = score.amax(dim=-1, keepdim=True)
            p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
            total_p = p.sum(dim=-1, keepdim=True)
            o = (p @ v) / torch.where(total_p > 0, total_p, torch.ones_like(total_p))
            out[at:at + n, h * group:(h + 1) * group] = o.transpose(0, 1).to(out.dtype)
        at += n
    return out


_RUN_PLAIN = {"quantize": _plain_quantize, "linear": _plain_linear, "append": _plain_append, "attend": _plain_attend}
_RUN_OWN = {"quantize": _own_quantize, "linear": _own_linear, "append": _own_append, "attend": _own_attend}


# ---------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"quantize": _exact_quantize, "linear": _exact_linear, "append": _exact_append, "attend": _exact_attend}[case["op"]](s)


def _exact_eighths(x, scale):
    """x / scale to the nearest whole number within [-127, 127]; the scale is the stored 32-bit one."""
    q = torch.zeros_like(x)
    ok = (scale > 0).expand_as(x)
    q[ok] = (x / scale.clamp_min(1e-300)).round().clamp(-127, 127)[ok]
    return q


def _exact_quantize(s):
    x = s["x"].double()
    scale = (x.abs().amax(dim=1, keepdim=True) / 127).float()
    return _exact_eighths(x, scale.double()) * scale, scale[:, 0]


def _exact_linear(s):
    x, out = s["x"], []
    w = s["w"].double() * s["ws"].double()[:, None]
    for rows in x.split(2048):
        r = rows.double()
        scale = (r.abs().amax(dim=1, keepdim=True) / 127).float().double()
        y = (_exact_eighths(r, scale) * scale) @ w.t()
        out.append(y if s["bias"] is None else y + s["bias"].double())
    return torch.cat(out)


def _exact_append(s):
    c = s["case"]
    page, rot, half = c["page"], c["rot"], c["rot"] // 2
    pair = [(2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half) for i in range(half)]
    one, two = [p[0] for p in pair], [p[1] for p in pair]

    def turn(x, first):
        """x [tokens, heads, d] at positions first, first + 1, ..."""
        y = x.double().clone()
        cos = s["cos"][first:first + len(x)].double()[:, None]
        sin = s["sin"][first:first + len(x)].double()[:, None]
        y[..., one] = x[..., one].double() * cos - x[..., two].double() * sin
        y[..., two] = x[..., two].double() * cos + x[..., one].double() * sin
        return y

    values = s["cache"].double() * s["scales"].double()[..., None, None]
    table = s["table"].tolist()
    q, at = [], 0
    for i, (n, old) in enumerate(zip(s["new"], s["prior"])):
        q.append(turn(s["q"][at:at + n], old))
        fresh = (turn(s["k"][at:at + n], old), s["v"][at:at + n].double())
        for first in range(old // page * page, old + n, page):
            slot = table[i][first // page]
            lo, hi = max(first, old), min(first + page, old + n)
            for side in (0, 1):
                x = fresh[side][lo - old:hi - old].transpose(0, 1)  # [heads, tokens, d]
                was = s["scales"][side, slot].double() if lo > first else torch.zeros(c["hkv"], dtype=torch.float64, device=x.device)
                now = torch.maximum(was, (x.abs().amax(dim=(1, 2)) / 127).float().double())[:, None, None]
                kept = s["cache"][side, slot, :, :lo - first].double()
                again = (kept * was[:, None, None] / now.clamp_min(1e-300)).round()
                values[side, slot, :, :lo - first] = torch.where(now > was[:, None, None], again, kept) * now
                values[side, slot, :, hi - first:] = s["cache"][side, slot, :, hi - first:].double() * now
                values[side, slot, :, lo - first:hi - first] = _exact_eighths(x, now) * now
        at += n
    return torch.cat(q), values


def _exact_attend(s):
    c = s["case"]
    group, d, page = c["hq"] // c["hkv"], c["d"], c["page"]
    if work(c)["flops"] > 6e12:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    at = 0
    for i, (n, old) in enumerate(zip(s["new"], s["prior"])):
        token = torch.arange(old + n, device=out.device)
        slot, offset = s["table"][i].long()[token // page], token % page
        for h in range(c["hkv"]):
            k = s["cache"][0, slot, h, offset].double() * s["scales"][0, slot, h].double()[:, None]
            v = s["cache"][1, slot, h, offset].double() * s["scales"][1, slot, h].double()[:, None]
            for lo in range(0, n, 512):  # queries in blocks, over the keys that the block can see
                hi = min(n, lo + 512)
                first = max(0, old + lo - c["window"] + 1) if c["window"] > 0 else 0
                last = old + hi
                q = s["q"][at + lo:at + hi, h * group:(h + 1) * group].double()
                score = torch.einsum("thd,kd->htk", q, k[first:last]) / math.sqrt(d)
                if c["cap"] > 0:
                    score = c["cap"] * torch.tanh(score / c["cap"])
                behind = (old + torch.arange(lo, hi, device=out.device))[:, None] - token[None, first:last]
                hidden = behind < 0
                if c["window"] > 0:
                    hidden |= behind >= c["window"]
                p = torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1)
                out[at + lo:at + hi, h * group:(h + 1) * group] = torch.einsum("htk,kd->thd", p, v[first:last])
        at += n
    return out
