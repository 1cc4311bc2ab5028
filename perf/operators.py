"""The paged-cache operators this package is measured on: what a program that serves several sequences from one pool of
key-value pages does per layer around its projections.

A case is a dict of plain values; `op` says which operator it calls:

  rotate    rotary positions of queries and keys: adjacent pairs or halves of the head, all or part of its channels, with
            the frequencies and the amplitude of a model stretched to long contexts; `grad`: with the gradients
  append    the keys and values of new tokens (one per sequence, or a ragged batch of chunks) go to their places in the
            paged cache; on the way the keys, and the queries beside them, are rotated
  attend    one new token per sequence attends to the sequence's paged cache, or to its last `window` tokens

A pool of pages is (n_kv_heads, n_pages, page_size, 2, head_dim): per token the key row, then the value row, as in the slot
table of the LRU cache.  Sequence b finds its token t in page `page_table[b, t // page_size]`.
"""

from __future__ import annotations

import math
import random

import torch

own = False   # True: `run` calls the package's operators; False: the plain form

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ELEMENT_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _rotate(name, batch, tokens, hq, hk, d, rot, dtype, interleaved, stretch=1.0, start=0, fused=False, grad=False):
    return {"name": name, "op": "rotate", "batch": batch, "tokens": tokens, "hq": hq, "hk": hk, "d": d, "rot": rot,
            "dtype": dtype, "interleaved": interleaved, "stretch": stretch, "start": start, "fused": fused, "grad": grad}


def _append(name, batch, new, hq, hk, d, rot, page, dtype, interleaved, before, spread, one=False, padding=0, stretch=1.0):
    return {"name": name, "op": "append", "batch": batch, "new": new, "hq": hq, "hk": hk, "d": d, "rot": rot, "page": page,
            "dtype": dtype, "interleaved": interleaved, "before": before, "spread": spread, "one": one, "padding": padding,
            "stretch": stretch}


def _attend(name, batch, length, spread, hk, rep, d, page, dtype, window=0, unused=0):
    return {"name": name, "op": "attend", "batch": batch, "length": length, "spread": spread, "hk": hk, "rep": rep, "d": d,
            "page": page, "dtype": dtype, "window": window, "unused": unused}


def listed():
    return [
        # the smallest rotation: the one new token of a 128K conversation
        _rotate("rotate-one-token", 1, 1, 32, 8, 128, 128, "bf16", True, start=131071),
        # two short prompts out of one fused projection, a third of the head rotated, positions squeezed four times
        _rotate("rotate-part-of-head-fused-fp16", 2, 2999, 12, 3, 96, 32, "fp16", False, stretch=4.0, fused=True),
        # a float32 notebook at positions near a million
        _rotate("rotate-1000-fp32", 1, 1000, 8, 2, 64, 64, "fp32", True, start=1000000),
        # fine-tuning on a stretched context: a 32K sequence, forward and backward
        _rotate("rotate-grad-32k", 1, 32768, 32, 8, 128, 128, "bf16", False, stretch=8.0, grad=True),
        # a decode step of 64 conversations
        _append("append-64-decode", 64, 1, 32, 8, 128, 128, 16, "bf16", True, before=5000, spread=4.0, one=True),
        # chunks of prompts of odd lengths, one sequence without a new token, a padded batch, pages of 24 tokens
        _append("append-chunks-fp16", 7, 700, 9, 3, 96, 48, 24, "fp16", False, before=900, spread=8.0, padding=37,
                stretch=2.0),
        # the prompt of a 32K document
        _append("append-32k", 1, 32768, 32, 8, 128, 128, 16, "bf16", True, before=0, spread=1.0),
        # the smallest attention: a float32 toy layer (tests, notebooks)
        _attend("attend-1-of-4k-fp32", 1, 4096, 1.0, 2, 4, 64, 16, "fp32"),
        # a layer with a sliding window, odd group and page sizes, two unused rows in the batch
        _attend("attend-9-windowed-fp16", 9, 6000, 6.0, 3, 5, 96, 24, "fp16", window=2000, unused=2),
        # batched serving: 64 conversations of a few thousand tokens
        _attend("attend-64-ragged", 64, 5000, 4.0, 8, 4, 128, 16, "bf16"),
        # one document of 128K tokens
        _attend("attend-1-of-128k", 1, 131072, 1.0, 8, 4, 128, 16, "bf16"),
        # a million tokens, one KV head: a GPU's share of a sharded model with sixteen queries to a key
        _attend("attend-1-of-1m-one-head", 1, 1048576, 1.0, 1, 16, 128, 32, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    e = ELEMENT_BYTES[dtype]
    d = rng.choice([64, 80, 96, 128, 128, 256])
    hk, rep = rng.randint(1, 8), rng.choice([1, 2, 3, 4, 4, 5, 6, 7, 8, 12, 16, 32])
    rot = rng.choice([d, d, d // 2, 16, 2 * rng.randint(1, d // 2)])
    page = rng.choice([1, 5, 8, 16, 16, 24, 32, 64, 100, 128])
    interleaved = rng.random() < 0.5
    stretch = rng.choice([1.0, 2.0, 8.0, 32.0])
    op = rng.choice(["rotate", "append", "attend", "attend"])
    if op == "rotate":
        batch = _log(rng, 1, 16)
        most = max(1, min(32768, int(5e8 / (2 * batch * hk * (rep + 1) * d * e))))
        return _rotate("", batch, _log(rng, 1, most), hk * rep, hk, d, rot, dtype, interleaved, stretch,
                       _log(rng, 1, 1000000), rng.random() < 0.3, rng.random() < 0.4)
    batch = _log(rng, 1, 256)
    if op == "append":
        one = rng.random() < 0.5
        most = max(1, min(32768, int(4e8 / (2 * batch * hk * (rep + 2) * d * e))))
        before = _log(rng, 1, max(1, min(100000, int(2e9 / (batch * hk * 2 * d * e)))))
        return _append("", batch, 1 if one else _log(rng, 1, most), hk * rep, hk, d, rot, page, dtype, interleaved,
                       before, rng.uniform(1.0, 8.0), one, rng.randint(0, 40) if not one else 0, stretch)
    most = max(2, min(1048576, int(8e8 / (batch * hk * 2 * d * e))))
    length = _log(rng, 1, most)
    return _attend("", batch, length, rng.uniform(1.0, 8.0), hk, rep, d, page, dtype,
                   rng.choice([0, 0, _log(rng, 1, max(2, length))]), rng.choice([0, 0, 1]) if batch > 1 else 0)


# ---- sizes that follow from a case --------------------------------------------------------

def _ragged(mean, spread, n, salt):
    """n lengths between mean / spread and mean * spread whose mean is near `mean`; the same for the same case."""
    if spread <= 1.0:
        return [mean] * n
    rng = random.Random(f"{mean} {spread:.6f} {n} {salt}")
    raw = [math.exp(rng.uniform(-math.log(spread), math.log(spread))) for _ in range(n)]
    scale = mean * n / sum(raw)
    return [max(1, int(round(r * scale))) for r in raw]


def _lengths(case):
    """attend: tokens in the cache per sequence, the new one among them; 0 for a row of the batch that is not in use"""
    out = _ragged(case["length"], case["spread"], case["batch"], "length")
    for i in range(case["unused"]):
        out[(i * 5 + 1) % case["batch"]] = 0
    return out


def _chunks(case):
    """append: (tokens cached before, new tokens) per sequence"""
    before = [b for b in _ragged(case["before"], case["spread"], case["batch"], "before")] if case["before"] else \
        [0] * case["batch"]
    if case["one"]:
        return before, [1] * case["batch"]
    new = _ragged(case["new"], case["spread"], case["batch"], "new")
    if case["batch"] > 2:
        new[2] = 0
    return before, new


def _attended(case):
    w = case["window"]
    return [min(n, w) if w else n for n in _lengths(case)]


def work(case):
    e, d = ELEMENT_BYTES[case["dtype"]], case["d"]
    if case["op"] == "attend":
        rows = case["batch"] * case["hk"] * case["rep"]
        n = sum(_attended(case))
        pages = sum(-(-a // case["page"]) for a in _attended(case))
        return {"bytes": n * case["hk"] * 2 * d * e + 2 * rows * d * e + 4 * pages,
                "flops": 4 * n * case["hk"] * case["rep"] * d}
    if case["op"] == "rotate":
        tokens, heads = case["batch"] * case["tokens"], case["hq"] + case["hk"]
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * tokens * heads * d * e + 4 * tokens), "flops": passes * 3 * tokens * heads * case["rot"]}
    tokens = sum(_chunks(case)[1])
    return {"bytes": 2 * tokens * (case["hq"] + 2 * case["hk"]) * d * e,
            "flops": 3 * tokens * (case["hq"] + case["hk"]) * case["rot"]}


# ---- inputs ---------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _frequencies(case):
    """base^(-2i/rot) as models keep them (float32), slowed for stretched contexts, and the amplitude that goes with it"""
    rot, stretch = case["rot"], case["stretch"]
    i = torch.arange(rot // 2, dtype=torch.float64)
    inv = 500000.0 ** (-2.0 * i / rot)
    if stretch > 1.0:
        ramp = ((i + 0.5) / (rot // 2)).clamp(0.0, 1.0)
        inv = inv * (1.0 - ramp) + inv / stretch * ramp
    return inv.to(torch.float32).cuda(), 1.0 + 0.1 * math.log(stretch)


def _heads(g, shape, dtype, outliers=True):
    """N(0,1) heads with a few channels that stand out"""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    if outliers:
        x[..., 3] *= 4.0
        x[..., shape[-1] // 2 + 1] *= 3.0
    return x.to(dtype)


def _table(g, counts, page, spare=2):
    """A page table over a shuffled pool: (batch, columns) int32, unused entries -1; pages in the pool"""
    pages = [-(-c // page) for c in counts]
    total = sum(pages) + spare
    ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(counts), max(pages + [1]) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, total


def prepare(case, seed):
    g = _gen(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] in ("rotate", "append"):
        s["inv_freq"], s["factor"] = _frequencies(case)
        if own:
            from dram_attention_b200 import Rotary
            s["rotary"] = Rotary(s["inv_freq"], factor=s["factor"], interleaved=case["interleaved"])
    if case["op"] == "rotate":
        shape = (case["batch"], case["tokens"])
        hq, hk, d = case["hq"], case["hk"], case["d"]
        if case["fused"]:
            qkv = _heads(g, shape + (hq + 2 * hk, d), dtype)
            s["q"], s["k"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
        else:
            s["q"], s["k"] = _heads(g, shape + (hq, d), dtype), _heads(g, shape + (hk, d), dtype)
        s["positions"] = (torch.arange(case["tokens"], device="cuda", dtype=torch.int32) + case["start"]).expand(shape)
        if case["grad"]:
            s["dq"], s["dk"] = _heads(g, shape + (hq, d), dtype, False), _heads(g, shape + (hk, d), dtype, False)
            s["q"], s["k"] = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
        return s
    hk, d, page = case["hk"], case["d"], case["page"]
    if case["op"] == "append":
        before, new = _chunks(case)
        after = [b + n for b, n in zip(before, new)]
        s["page_table"], n_pages = _table(g, after, page)
        s["lengths"] = torch.tensor(after, dtype=torch.int32, device="cuda")
        s["starts_host"] = [sum(new[:i]) for i in range(len(new) + 1)]
        s["starts"] = torch.tensor(s["starts_host"], dtype=torch.int32, device="cuda")
        s["before_host"] = before
        rows = sum(new) + case["padding"]
        s["q"], s["k"] = _heads(g, (rows, case["hq"], d), dtype), _heads(g, (rows, hk, d), dtype)
        s["v"] = _heads(g, (rows, hk, d), dtype, False)
        s["pages"] = torch.randn((hk, n_pages, page, 2, d), generator=g, device="cuda").to(dtype)
        if own:
            from dram_attention_b200 import PagedKVCache
            s["cache"] = PagedKVCache.over(s["pages"])
        return s
    lengths = _lengths(case)
    s["page_table"], n_pages = _table(g, lengths, page)
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["lengths_host"] = lengths
    pages = torch.empty((hk, n_pages, page, 2, d), dtype=dtype, device="cuda")
    for h in range(hk):
        pages[h] = _heads(g, (n_pages, page, 2, d), dtype)
    # a few pages whose keys lie along a direction that the queries share
    needle = torch.randn((hk, 1, 1, d), generator=g, device="cuda")
    marked = torch.randint(n_pages, (max(1, n_pages // 64),), generator=g, device="cuda")
    pages[:, marked, :, 0] = (pages[:, marked, :, 0].float() + 0.5 * needle).to(dtype)
    s["pages"] = pages
    q = torch.randn((case["batch"], hk, case["rep"], d), generator=g, device="cuda") + 0.5 * needle[:, 0]
    s["q"] = q.reshape(case["batch"], hk * case["rep"], d).to(dtype)
    if own:
        from dram_attention_b200 import PagedKVCache
        s["cache"] = PagedKVCache.over(pages)
    return s


# ---- plain forms ------------------------------------------------------------------------------

def _rotate_plain(x, positions, inv_freq, factor, interleaved):
    """x (..., heads, d) float32, positions (...)"""
    rot = 2 * inv_freq.numel()
    angle = positions.double()[..., None] * inv_freq.double()
    cos, sin = (angle.cos() * factor).float()[..., None, :], (angle.sin() * factor).float()[..., None, :]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    return y


def _run_rotate(s):
    case = s["case"]
    q, k, positions = s["q"], s["k"], s["positions"]
    if own:
        q2, k2 = s["rotary"](q, k, positions)
        if not case["grad"]:
            return q2, k2
        return (q2.detach(), k2.detach()) + torch.autograd.grad((q2, k2), (q, k), (s["dq"], s["dk"]))
    turn = (positions, s["inv_freq"], s["factor"], case["interleaved"])
    out = [_rotate_plain(x.detach().float(), *turn).to(x.dtype) for x in (q, k)]
    if case["grad"]:   # a rotation's gradient is the rotation back, with the same amplitude
        back = (-positions, s["inv_freq"], s["factor"], case["interleaved"])
        out += [_rotate_plain(x.float(), *back).to(x.dtype) for x in (s["dq"], s["dk"])]
    return tuple(out)


def _run_append(s):
    case = s["case"]
    page, one = case["page"], case["one"]
    if own:
        q = s["cache"].append_(s["k"], s["v"], s["page_table"], s["lengths"], starts=None if one else s["starts"], q=s["q"],
                               rotary=s["rotary"])
        return q, s["pages"]
    # token by token: its sequence, its position, its place in the pool
    total = s["starts_host"][-1]
    tokens = torch.arange(total, device="cuda")
    seq = torch.searchsorted(s["starts"].long(), tokens, right=True) - 1
    new = s["starts"][1:] - s["starts"][:-1]
    position = (s["lengths"] - new)[seq].long() + tokens - s["starts"][seq]
    where = s["page_table"][seq, position // page].long()
    turn = (position, s["inv_freq"], s["factor"], case["interleaved"])
    k = _rotate_plain(s["k"][:total].float(), *turn).to(s["k"].dtype)
    s["pages"][:, where, position % page, 0] = k.transpose(0, 1)
    s["pages"][:, where, position % page, 1] = s["v"][:total].transpose(0, 1)
    q = torch.zeros_like(s["q"])   # rows behind the last sequence stay zero
    q[:total] = _rotate_plain(s["q"][:total].float(), *turn).to(q.dtype)
    return q, s["pages"]


def _run_attend(s):
    case = s["case"]
    hk, rep, d, page, window = case["hk"], case["rep"], case["d"], case["page"], case["window"]
    if own:
        return s["cache"].attend(s["q"], s["page_table"], s["lengths"], window=window)
    out = torch.zeros_like(s["q"])
    for b, n in enumerate(s["lengths_host"]):
        if n == 0:
            continue
        first = max(0, n - window) if window else 0
        p0 = first // page
        ids = s["page_table"][b, p0:-(-n // page)].long()
        kv = s["pages"][:, ids].reshape(hk, -1, 2, d)[:, first - p0 * page:n - p0 * page].float()
        q = s["q"][b].float().reshape(hk, rep, d)
        score = q @ kv[:, :, 0].transpose(1, 2) / math.sqrt(d)
        weight = torch.exp(score - score.amax(-1, keepdim=True))
        out[b] = (weight @ kv[:, :, 1] / weight.sum(-1, keepdim=True)).reshape(hk * rep, d).to(out.dtype)
    return out


def run(state):
    return {"rotate": _run_rotate, "append": _run_append, "attend": _run_attend}[state["case"]["op"]](state)


# ---- from the definitions, in 64 bits -----------------------------------------------------------

def _turned(x, positions, inv_freq, factor, interleaved):
    """The definition as a product of complex numbers: channel pairs times factor * exp(i * position * frequency)"""
    x = x.detach().double()
    half = inv_freq.numel()
    w = torch.polar(torch.full((), factor, dtype=torch.float64, device=x.device),
                    positions.double().unsqueeze(-1) * inv_freq.double()).unsqueeze(-2)
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    pairs = head.unflatten(-1, (half, 2)) if interleaved else head.unflatten(-1, (2, half)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * w)
    z = z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)
    return torch.cat([z, rest], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        how = (s["inv_freq"], s["factor"], case["interleaved"])
        out = [_turned(s[n], s["positions"], *how) for n in ("q", "k")]
        if case["grad"]:
            out += [_turned(s[n], -s["positions"], *how) for n in ("dq", "dk")]
        return tuple(out)
    if case["op"] == "append":
        pages, q = s["pages"].double(), torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        how = (s["inv_freq"], s["factor"], case["interleaved"])
        for b, before in enumerate(s["before_host"]):
            lo, hi = s["starts_host"][b], s["starts_host"][b + 1]
            if lo == hi:
                continue
            position = before + torch.arange(hi - lo, device="cuda")
            slot = s["page_table"][b].long()[position // case["page"]] * case["page"] + position % case["page"]
            flat = pages.flatten(1, 2)
            flat[:, slot, 0] = _turned(s["k"][lo:hi], position, *how).transpose(0, 1)
            flat[:, slot, 1] = s["v"][lo:hi].double().transpose(0, 1)
            q[lo:hi] = _turned(s["q"][lo:hi], position, *how)
        return q, pages
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    rep = case["rep"]
    for b, n in enumerate(s["lengths_host"]):
        token = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device="cuda")
        if n == 0:
            continue
        place = s["page_table"][b].long()[token // case["page"]]
        for h in range(case["hk"]):
            rows = s["pages"][h][place, token % case["page"]].double()
            score = s["q"][b, h * rep:(h + 1) * rep].double() @ rows[:, 0].T * case["d"] ** -0.5
            out[b, h * rep:(h + 1) * rep] = torch.softmax(score, -1) @ rows[:, 1]
    return out
