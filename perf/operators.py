"""What the paged key-value cache's operators are measured on.

Three operators of a decode step: ``write`` stores new keys and values in a paged cache
(rounded to the cache's type, or quantised to 8 bits with one scale per token and head),
``read`` gathers them back, and ``attend`` is the attention of one new token per
sequence over the cache. With ``own`` false they are computed in plain tensor
operations; with ``own`` true by this package's operators.

A cache is ``[pages, page_size, kv_heads, head_dim]``; token ``t`` of sequence ``b`` is in
slot ``tables[b, t // page_size] * page_size + t % page_size``.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8,
          "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "e4m3": 1}
CODE_MAX = {"i8": 127.0, "e4m3": 448.0}


# -- cases -------------------------------------------------------------------------------


def _attend(name, batch, heads, kv_heads, dim, page, shortest, longest, q, cache, window=0, empty=0, lse=False):
    """``batch`` sequences of lengths between ``shortest`` and ``longest`` (both met),
    the last ``empty`` of them of length zero (a padded batch)."""
    return {"name": name, "op": "attend", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "shortest": shortest, "longest": longest, "q": q, "cache": cache, "window": window,
            "empty": empty, "lse": lse}


def _rows(name, op, tokens, kv_heads, dim, page, x, cache, skipped=0, fused=False):
    """``tokens`` rows written or read, the last ``skipped`` of them padding (slot -1);
    ``fused``: k and v are slices of one projection's output."""
    return {"name": name, "op": op, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "page": page, "x": x,
            "cache": cache, "skipped": skipped, "fused": fused}


def listed():
    return [
        # one user, a short prompt: every call is latency
        _attend("attend one short", 1, 32, 8, 128, 16, 100, 100, "bf16", "bf16"),
        # a batch of chats of very different lengths
        _attend("attend chats", 16, 32, 8, 128, 16, 37, 4001, "bf16", "bf16"),
        # a full server: the largest batch, long sequences
        _attend("attend full", 64, 32, 8, 128, 16, 4096, 8192, "bf16", "bf16"),
        # one user with a book in the prompt: the length itself has to be split
        _attend("attend one long", 1, 32, 8, 128, 16, 120001, 120001, "bf16", "bf16", lse=True),
        # a program of this framework: fp32 throughout, 128 heads of 64, 1024 tokens
        _attend("attend fp32", 8, 16, 16, 64, 32, 1024, 1024, "f32", "f32"),
        # an fp32 program over an 8-bit cache, grouped heads
        _attend("attend int8", 32, 32, 4, 64, 16, 500, 6000, "f32", "i8"),
        # a long-context server with an 8-bit cache, a sliding window and a padded batch
        _attend("attend e4m3 window", 48, 64, 8, 128, 64, 1, 9000, "bf16", "e4m3", window=4096, empty=3),
        # one key-value head for all query heads, wide heads, odd lengths
        _attend("attend shared head", 7, 16, 1, 256, 8, 777, 20011, "f16", "f16", lse=True),
        # every decode step: one token a sequence
        _rows("write step", "write", 16, 8, 128, 16, "bf16", "e4m3"),
        # a prompt's chunk, straight from the fused projection of an fp32 program
        _rows("write prompt", "write", 16384, 8, 128, 16, "f32", "i8", skipped=100, fused=True),
        # reading a prefix back for the next chunk of a prompt
        _rows("read prefix", "read", 24577, 8, 128, 16, "f32", "i8"),
        # looking at a short prefix in an 8-bit cache
        _rows("read short", "read", 333, 4, 64, 16, "bf16", "e4m3", skipped=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["attend", "attend", "attend", "write", "read"])
    cache = rng.choice(["f32", "f16", "bf16", "i8", "e4m3"])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
    dim = rng.choice([32, 64, 80, 96, 128, 128, 256])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    if kind != "attend":
        x = cache if cache in ("f16", "bf16") and rng.random() < 0.5 else rng.choice(["f32", "f16", "bf16"])
        tokens = _log(rng, 1, (1 << 25) // (kv_heads * dim))
        case = _rows("", kind, tokens, kv_heads, dim, page, x, cache, rng.choice([0, 0, tokens // 7]),
                     kind == "write" and rng.random() < 0.3)
    else:
        q = {"f32": ["f32"], "f16": ["f16", "f32"], "bf16": ["bf16", "f32"]}.get(cache, ["f32", "f16", "bf16"])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 4, 5, 8, 16])
        batch = _log(rng, 1, 192)
        token = kv_heads * dim * 2 * max(2, BYTES[cache])  # a token's bytes, 8-bit ones counted as 16
        longest = _log(rng, 1, max(2, min(131072, (1 << 30) // (token * batch))))
        shortest = rng.randint(1, longest)
        case = _attend("", batch, heads, kv_heads, dim, page, shortest, longest, rng.choice(q), cache,
                       rng.choice([0, 0, 0, max(1, longest // 3)]), rng.choice([0, 0, batch // 5]),
                       rng.random() < 0.3)
    del case["name"]
    return case


def _lengths(case):
    """The sequences' lengths: part of a case, not of its seed, so that its work is known."""
    rng = random.Random(case["batch"] * 1000003 + case["longest"])
    n = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]
    n[0] = case["longest"]
    if case["batch"] > 1:
        n[-1] = case["shortest"]
    rng.shuffle(n)
    return n[: case["batch"] - case["empty"]] + [0] * case["empty"]


def _visible(case):
    return sum(min(n, case["window"]) if case["window"] else n for n in _lengths(case))


def work(case):
    c, d, hk = BYTES[case["cache"]], case["dim"], case["kv_heads"]
    scale = 4 if case["cache"] in CODE_MAX else 0
    if case["op"] == "attend":
        q, b = BYTES[case["q"]], case["batch"]
        n = _visible(case)
        tables = 4 * sum(-(-x // case["page"]) for x in _lengths(case)) + 4 * b
        return {"bytes": n * hk * 2 * (d * c + scale) + b * case["heads"] * (2 * d * q + 4 * case["lse"]) + tables,
                "flops": 4 * n * case["heads"] * d}
    n = case["tokens"] - case["skipped"]
    return {"bytes": n * hk * 2 * (d * (c + BYTES[case["x"]]) + scale) + 8 * case["tokens"],
            "flops": 4 * n * hk * d}


# -- inputs ------------------------------------------------------------------------------


def _cache(case, pages, g):
    """A cache that earlier steps have filled: (k_cache, v_cache, k_scale, v_scale)."""
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    kind = case["cache"]
    filled = []
    for _ in range(2):
        x = torch.randn(shape, generator=g, device="cuda")
        if kind == "i8":
            x = (x * 40.0).round_().clamp_(-127, 127)
        elif kind == "e4m3":
            x = (x * 120.0).clamp_(-448, 448)
        filled.append(x.to(DTYPES[kind]))
        del x
    if kind not in CODE_MAX:
        return filled[0], filled[1], None, None
    spread = 0.025 if kind == "i8" else 0.008
    scales = [(0.3 + 1.4 * torch.rand(shape[:3], generator=g, device="cuda")) * spread for _ in range(2)]
    return filled[0], filled[1], scales[0], scales[1]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    page = case["page"]
    if case["op"] == "attend":
        lengths = _lengths(case)
        used = [-(-n // page) for n in lengths]
        width = max(1, max(used))
        pages = sum(used) + 3
        order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32).cpu()
        tables = torch.full((case["batch"], width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(used):
            tables[b, :n] = order[at:at + n]
            at += n
        k, v, ks, vs = _cache(case, pages, g)
        q = torch.randn((case["batch"], case["heads"], case["dim"]), generator=g, device="cuda")
        q = (q * (1.0 + 2.0 * torch.rand((case["batch"], case["heads"], 1), generator=g, device="cuda")))
        return {"case": case, "q": q.to(DTYPES[case["q"]]), "k_cache": k, "v_cache": v, "k_scale": ks, "v_scale": vs,
                "tables": tables.cuda(), "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                "scale": 1.0 / math.sqrt(case["dim"])}
    n = case["tokens"]
    pages = -(-n // page) + 5
    k, v, ks, vs = _cache(case, pages, g)
    # whole pages in a random order, tokens in order within each: what an allocator hands out
    order = torch.randperm(pages, generator=g, device="cuda")[: -(-n // page)]
    slots = (order[:, None] * page + torch.arange(page, device="cuda")[None, :]).reshape(-1)[:n].contiguous()
    if case["skipped"]:
        slots[n - case["skipped"]:] = -1
    state = {"case": case, "k_cache": k, "v_cache": v, "k_scale": ks, "v_scale": vs, "slots": slots}
    if case["op"] == "write":
        parts = 4 if case["fused"] else 2
        x = torch.randn((n, parts, case["kv_heads"], case["dim"]), generator=g, device="cuda")
        x *= 0.2 + 2.0 * torch.rand((1, parts, case["kv_heads"], case["dim"]), generator=g, device="cuda")
        x = x.to(DTYPES[case["x"]])
        state["new_k"], state["new_v"] = (x[:, -2], x[:, -1]) if case["fused"] else (x[:, 0].contiguous(), x[:, 1].contiguous())
    return state


# -- the operators, plain ----------------------------------------------------------------


def _codes(x, kind):
    """(codes, scales) of rows ``x`` (..., head_dim): the scale is the row's largest
    magnitude over the largest code, in fp32; a code is the nearest to x / scale, ties to
    even. The quotient is taken in 64 bits: in 32 it can be rounded onto a border."""
    largest = x.float().abs().amax(-1)
    scale = largest / torch.full_like(largest, CODE_MAX[kind])  # by a tensor: a true division
    t = x.double() / torch.where(scale > 0, scale, 1.0).double().unsqueeze(-1)
    if kind == "i8":
        return t.round().to(torch.int8), scale
    # 2**exponent of t, exactly: t over its fraction; e4m3 keeps 3 bits behind the leading one, 2**-9 at least
    power = torch.where(t == 0, 1.0, t / torch.where(t == 0, 1.0, torch.frexp(t)[0]))
    step = power.clamp(min=2.0 ** -5) / 16.0
    return ((t / step).round() * step).float().to(torch.float8_e4m3fn), scale


def _stored(x, kind):
    """8-bit types as bytes: indexed stores of the others need no care."""
    return x.view(torch.uint8) if kind in CODE_MAX else x


def _plain_write(s):
    kind = s["case"]["cache"]
    keep = s["slots"] >= 0
    slots = s["slots"][keep]
    for x, cache, scales in ((s["new_k"], s["k_cache"], s["k_scale"]), (s["new_v"], s["v_cache"], s["v_scale"])):
        if scales is not None:
            codes, scale = _codes(x[keep], kind)
            scales.view(-1, scales.shape[2])[slots] = scale
        else:
            codes = x[keep].to(cache.dtype)
        _stored(cache, kind).view((-1,) + cache.shape[2:])[slots] = _stored(codes, kind)


def _plain_read(s):
    case, out = s["case"], []
    ok = (s["slots"] >= 0)[:, None, None]
    slots = s["slots"].clamp(min=0)
    for cache, scales in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])):
        x = _stored(cache, case["cache"]).view((-1,) + cache.shape[2:])[slots]
        x = x.view(cache.dtype).float()
        if scales is not None:
            x = x * scales.view(-1, scales.shape[2])[slots].unsqueeze(-1)
        out.append(torch.where(ok, x, 0.0).to(DTYPES[case["x"]]))
    return out


def _dense(cache, scales, kind, tables):
    """The sequences' rows side by side in 32 bits: (batch, tokens, kv_heads, head_dim)."""
    at = tables.clamp(min=0).long()
    x = _stored(cache, kind)[at]
    x = x.view(cache.dtype).float()
    if scales is not None:
        x *= scales[at].unsqueeze(-1)
    return x.flatten(1, 2)


def _plain_attend(s):
    case = s["case"]
    b, h, d = s["q"].shape
    hk = case["kv_heads"]
    n = s["lengths"].long()[:, None]
    t = torch.arange(s["tables"].shape[1] * case["page"], device="cuda")[None, :]
    seen = (t < n) & (t >= n - case["window"]) if case["window"] else t < n
    k = _dense(s["k_cache"], s["k_scale"], case["cache"], s["tables"])
    q = s["q"].float().view(b, hk, h // hk, d)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)) * s["scale"]
    del k
    scores.masked_fill_(~seen[:, None, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = _dense(s["v_cache"], s["v_scale"], case["cache"], s["tables"])
    o = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, 1.0)
    out = o.reshape(b, h, d).to(s["q"].dtype)
    return (out, (top + torch.log(total)).reshape(b, h)) if case["lse"] else out


# -- one pass ----------------------------------------------------------------------------


def run(state):
    case = state["case"]
    scales = {"k_scale": state["k_scale"], "v_scale": state["v_scale"]}
    if case["op"] == "attend":
        if own:
            import metellus_b200

            return metellus_b200.paged_attention(state["q"], state["k_cache"], state["v_cache"], state["tables"],
                                                 state["lengths"], scale=state["scale"], window=case["window"],
                                                 return_lse=case["lse"], **scales)
        return _plain_attend(state)
    if case["op"] == "read":
        if own:
            import metellus_b200

            return metellus_b200.cache_read(state["k_cache"], state["v_cache"], state["slots"],
                                            dtype=DTYPES[case["x"]], **scales)
        return _plain_read(state)
    if own:
        import metellus_b200

        metellus_b200.cache_write(state["new_k"], state["new_v"], state["k_cache"], state["v_cache"], state["slots"],
                                  **scales)
    else:
        _plain_write(state)
    # the updated cache itself; the 8-bit codes are numbers of their type
    return [state["k_cache"], state["v_cache"]] + [x for x in scales.values() if x is not None]


# -- the definition in 64 bits -------------------------------------------------------------


def _values(cache, scales):
    x = cache.double()
    return x if scales is None else x * scales.double()[..., None]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["cache"]
    if case["op"] == "attend":
        g, page = case["heads"] // case["kv_heads"], case["page"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
        for b, n in enumerate(_lengths(case)):
            if n == 0:
                continue
            ids = s["tables"][b, : -(-n // page)].long()
            lo = max(0, n - case["window"]) if case["window"] else 0
            first = lo // page
            ids = ids[first:]
            take = slice(lo - first * page, n - first * page)
            k, v = (_values(c.view(torch.uint8)[ids].view(c.dtype) if kind in CODE_MAX else c[ids],
                            None if z is None else z[ids]).flatten(0, 1)[take]
                    for c, z in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))
            q = s["q"][b].double().unflatten(0, (case["kv_heads"], g))
            scores = torch.einsum("hgd,thd->hgt", q, k) * s["scale"]
            lse[b] = torch.logsumexp(scores, -1).flatten()
            out[b] = torch.einsum("hgt,thd->hgd", torch.softmax(scores, -1), v).flatten(0, 1)
        return (out, lse) if case["lse"] else out
    keep = s["slots"] >= 0
    slots = s["slots"][keep]
    pairs = ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"]))
    if case["op"] == "read":
        got = []
        for c, z in pairs:
            y = torch.zeros((case["tokens"], case["kv_heads"], case["dim"]), dtype=torch.float64, device="cuda")
            y[keep] = _values(c, z).flatten(0, 1)[slots]
            got.append(y)
        return got
    caches, scales = [], []
    for x, (c, z) in zip((s["new_k"], s["new_v"]), pairs):
        x = x[keep].double()
        c = c.double().flatten(0, 1)
        if z is not None:
            z = z.double().flatten(0, 1)
            z[slots] = x.abs().amax(-1) / CODE_MAX[kind]
            # the stored scale is the fp32 one: the codes are quotients by it
            x = x / z[slots].float().double().clamp(min=1e-300)[..., None]
            scales.append(z.unflatten(0, (-1, case["page"])))
        c[slots] = x
        caches.append(None if kind == "i8" else c.unflatten(0, (-1, case["page"])))
    return caches + scales
