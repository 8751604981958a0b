"""Plain 64-bit forms of the paged cache's operators, on whatever device the arrays are,
and the tolerances of their tests (derived, not fitted).

Attention. Let u(t) = finfo(t).eps / 2 be the rounding of type t. Errors of an output o =
sum p v / sum p, with A = sum p |v| / sum p:

* scores: a dot product of D terms in fp32, rounded to nearest or truncated (an ulp,
  2^-23), errs by at most (D + 8) 2^-23 sum |q k|; times the scale, plus a few roundings of
  the score itself on the way to exp2. A score off by ds scales its p by exp(ds): the output
  moves by at most 2 ds A (numerator and denominator) while ds is small;
* probabilities rounded to the product's operand type: u(p) A;
* sums over n tokens in fp32: n 2^-23 A each for numerator and denominator;
* probabilities too small for their type: each loses at most half its smallest step, at most
  2^-36 of the largest one where operands are fp16 (held times at least 2^11, smallest step
  2^-24), 2^-126 in the others' range; that is n 2^-36 (or n 2^-126) times the largest value a row of V
  can hold (scale times largest code, as scales are multiplied in with them);
* the output's own rounding: u(out) |o|, at least half its type's smallest step.

Operands of 32 bits are split into pieces that together keep at least 22 bits: 2^-21 A, and
2^-21 sum |q k| in the scores."""

from __future__ import annotations

import math

import torch

CODE_MAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def half_step(t: torch.dtype) -> float:
    return torch.finfo(t).eps / 2


def values(cache, scale=None):
    x = cache.double()
    return x if scale is None else x * scale.double()[..., None]


def codes(x, dtype):
    """(codes as float64, float32 scales) of rows (..., head_dim)."""
    big = x.float().abs().amax(-1)
    scale = big / torch.full_like(big, CODE_MAX[dtype])
    finite = torch.isfinite(x.float()).all(-1)
    scale = torch.where(finite, scale, torch.full_like(scale, math.nan))
    ok = finite & (scale > 0)
    t = torch.where(ok[..., None], x.double() / torch.where(ok, scale, torch.ones_like(scale)).double()[..., None], 0.0)
    if dtype is torch.int8:
        return t.round().clamp(-127, 127), scale
    exponent = torch.floor(torch.log2(t.abs().clamp(min=1e-30))).clamp(min=-6)
    step = torch.exp2(exponent - 3)
    return (t / step).round() * step, scale


def attention(q, k_cache, v_cache, tables, lengths, *, k_scale=None, v_scale=None, scale=None, window=0):
    """(out, lse, tol): all in float64; tol is the per-element tolerance."""
    b, h, d = q.shape
    pages, ps, hk, _ = k_cache.shape
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros((b, h, d), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    lse = torch.full((b, h), -math.inf, dtype=torch.float64, device=q.device)
    lse_tol = torch.zeros_like(lse)
    K = values(k_cache, k_scale)
    V = values(v_cache, v_scale)
    split = q.dtype == torch.float32
    operand = torch.float16 if k_cache.dtype in CODE_MAX else k_cache.dtype
    up = 2.0 ** -21 if split else half_step(operand)
    lost = 2.0 ** -36 if operand is torch.float16 else 2.0 ** -126
    least = torch.finfo(q.dtype).smallest_normal * half_step(q.dtype)
    for i in range(b):
        n = min(max(int(lengths[i]), 0), tables.shape[1] * ps)
        t = torch.arange(max(0, n - window) if window else 0, n, device=q.device)
        page = tables[i].long()[t // ps] if n else t
        t, page = t[(page >= 0) & (page < pages)], page[(page >= 0) & (page < pages)]
        if t.numel() == 0:
            continue
        k, v = K[page, t % ps], V[page, t % ps]
        qi = q[i].double().unflatten(0, (hk, h // hk))
        s = torch.einsum("hgd,thd->hgt", qi, k) * scale
        p = torch.softmax(s, -1)
        lse[i] = torch.logsumexp(s, -1).flatten()
        o = torch.einsum("hgt,thd->hgd", p, v)
        size = torch.einsum("hgd,thd->hgt", qi.abs(), k.abs()).nan_to_num(0, 0, 0).amax(-1) * abs(scale)
        ds = size * ((d + 8) * 2.0 ** -23 + (2.0 ** -21 if split else 0)) + 4 * 2.0 ** -23 * size
        A = torch.einsum("hgt,thd->hgd", p, v.abs())
        n_err = 2 * (t.numel() + 16) * 2.0 ** -23
        largest = v.abs().nan_to_num(0, 0, 0).amax()
        if v_scale is not None:
            largest = v_scale[page, t % ps].double().nan_to_num(0, 0, 0).amax() * CODE_MAX[v_cache.dtype]
        out[i] = o.flatten(0, 1)
        tol[i] = (A * (up + n_err + 2 * ds[..., None]) * 1.01 + half_step(q.dtype) * o.abs()
                  + t.numel() * lost * largest + least).flatten(0, 1)
        lse_tol[i] = (ds + n_err + 4 * 2.0 ** -23 * lse[i].abs().unflatten(0, (hk, h // hk))).flatten() + 2.0 ** -22
    return out, lse, tol, lse_tol


def check(got, want, tol, what=""):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaNs differ"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    ok = torch.isfinite(want)
    err, tol = (got - want).abs()[ok], tol[ok]
    if err.numel() and not bool((err <= tol).all()):
        i = int((err - tol).argmax())
        raise AssertionError(f"{what}: error {err[i]:.3e} over tolerance {tol[i]:.3e} (value {want[ok][i]:.6e}); "
                             f"{int((err > tol).sum())} of {err.numel()} outside")
