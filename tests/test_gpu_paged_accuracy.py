"""How near the paged attention's outputs are to the formula in 64 bits, where the bounds of
``paged_reference`` are too wide to show it: every output must be what some number within the
kernel's own error of the exact one rounds to.

That error, with D terms a score, n tokens and A = sum p |v|:

* scores: (D + 12) 2^-23 sum |q k|, and D 2^-24 max |q| max |k| where elements of a query are held
  as multiples of 2^-24 of its largest; a score off by ds moves an output by 2 ds A;
* exponentials, products and sums: 2 (n + 16) 2^-23 A;
* probabilities in two pieces, of half a step each: 2^-22 A (fp16), 2^-16 A (bf16), and, of fp16, half
  the smallest step: 2^-35 of the largest weight that a token has (2^-29 where a weight is a product with a
  scale of V), times the largest V, n times."""

from __future__ import annotations

import pytest
import torch

from metellus_b200 import paged_attention

pytestmark = pytest.mark.gpu

F32, F16, BF16, I8, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn
DEV = "cuda"


@pytest.fixture(autouse=True)
def _device(cuda_device):
    torch.manual_seed(7)


def attend(q, k, v, n, k_scale=None, v_scale=None):
    """The kernel's outputs for caches given as rows [batch, tokens, kv_heads, dim], in pages of 8."""
    b, tokens = k.shape[:2]
    k, v, k_scale, v_scale = (None if x is None else x.unflatten(1, (-1, 8)).flatten(0, 1) for x in (k, v, k_scale, v_scale))
    tables = torch.arange(b * tokens // 8, device=DEV, dtype=torch.int32).view(b, -1)
    return paged_attention(q, k, v, tables, n, k_scale=k_scale, v_scale=v_scale)


def exact(q, k, v, n, k_scale=None, v_scale=None):
    """(outputs, error before they are rounded), float64."""
    b, heads, dim = q.shape
    piece = 2.0 ** -16 if k.dtype is BF16 else 2.0 ** -22
    one = torch.ones(k.shape[:3], device=DEV, dtype=torch.float64)
    ks, vs = (one if z is None else z.double() for z in (k_scale, v_scale))
    codes, k, v = v.double(), k.double() * ks[..., None], v.double() * vs[..., None]
    q = q.double().unflatten(1, (k.shape[2], -1))
    there = (torch.arange(k.shape[1], device=DEV) < n[:, None])[:, None, None, :]
    s = torch.einsum("bhgd,bthd->bhgt", q, k) * dim ** -0.5
    p = torch.softmax(s.masked_fill(~there, -torch.inf), -1)
    size = torch.einsum("bhgd,bthd->bhgt", q.abs(), k.abs()).masked_fill(~there, 0).amax(-1, keepdim=True)
    least = q.abs().amax(-1, keepdim=True) * k.abs().amax((1, 3))[:, :, None, None]
    ds = ((dim + 12) * 2.0 ** -23 * size + dim * 2.0 ** -24 * least) * dim ** -0.5
    o = torch.einsum("bhgt,bthd->bhgd", p, v)
    A = torch.einsum("bhgt,bthd->bhgd", p, v.abs())
    weight = (p * vs.transpose(1, 2)[:, :, None, :]).amax(-1, keepdim=True)
    d = A * (piece + 2 * ds + 2 * (n.double()[:, None, None, None] + 16) * 2.0 ** -23)
    d = d + n[:, None, None, None] * 2.0 ** (-35 if v_scale is None else -29) * weight * codes.abs().amax()
    return o.flatten(1, 2), d.flatten(1, 2)


def check(got, o, d):
    lo, hi = (o - d).to(got.dtype), (o + d).to(got.dtype)
    bad = ~((lo <= got) & (got <= hi))
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} outside, such as {got[bad][0]:.9g} of "
                           f"{lo[bad][0]:.9g} .. {hi[bad][0]:.9g}")


def codes(shape, dtype):
    return (torch.randn(shape, device=DEV) * 30).round().clamp(-100, 100).to(dtype)


@pytest.mark.parametrize("q_type,dtype", [(BF16, I8), (BF16, E4M3), (F16, I8), (F16, E4M3), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (16, 1, 80)])
def test_probabilities_keep_their_bits(q_type, dtype, heads, kv_heads, dim):
    """A few tokens of about equal weight: one rounded piece a probability would show in the outputs."""
    shape = (96, 8, kv_heads, dim)
    scaled = dtype in (I8, E4M3)
    k, v = (codes(shape, dtype) if scaled else torch.randn(shape, device=DEV).to(dtype) for _ in range(2))
    z = [0.002 + 0.03 * torch.rand(shape[:3], device=DEV) if scaled else None for _ in range(2)]
    q = (torch.randn((shape[0], heads, dim), device=DEV) * 0.3).to(q_type)
    n = torch.randint(2, 9, (shape[0],), device=DEV, dtype=torch.int32)
    check(attend(q, k, v, n, *z), *exact(q, k, v, n, *z))


@pytest.mark.parametrize("q_type,dtype", [(F16, F16), (BF16, BF16), (F16, E4M3), (F32, F16), (F32, F32)])
def test_long_sums_do_not_drift(q_type, dtype):
    """Values of one sign, thousands of tiles a warp, in a cache of 512 tokens that is seen 256 times over. Outputs
    are, on the average, what the exact ones round to: a shift of them by 2^-15, a sixteenth of fp16's half step,
    moves that many more to the next value. (Not the mean of their errors: the 1024 values differ little from
    one sequence to another, so bf16's roundings alone have a mean of 2^-8 / sqrt(3 * 1024).)"""
    batch, heads, kv_heads, dim, tokens, times = 32, 32, 8, 128, 512, 256
    k = torch.randn((1, tokens, kv_heads, dim), device=DEV).to(dtype)
    v = (1 + 0.2 * torch.randn((1, tokens, kv_heads, dim), device=DEV)).to(dtype)
    q = (torch.randn((batch, heads, dim), device=DEV) * 0.25).to(q_type)
    z = [torch.ones((1, tokens, kv_heads), device=DEV) if dtype is E4M3 else None] * 2
    pages = [None if x is None else x.unflatten(1, (-1, 8)).flatten(0, 1) for x in (k, v, *z)]
    tables = torch.arange(tokens // 8, device=DEV, dtype=torch.int32).repeat(batch, times)
    n = torch.full((batch,), tokens * times, device=DEV, dtype=torch.int32)
    got = paged_attention(q, *pages[:2], tables, n, k_scale=pages[2], v_scale=pages[3]).double()
    seen = torch.full((batch,), tokens, device=DEV, dtype=torch.int32)
    o, _ = exact(q, *(x.expand(batch, -1, -1, -1) for x in (k, v)), seen, *(None if x is None else x.expand(batch, -1, -1) for x in z))
    assert abs(float(((got - o.to(q_type).double()) / o).mean())) <= 2.0 ** -15
    half_step = torch.finfo(q_type).eps / 2
    assert float(((got - o) / o).abs().max()) <= half_step + 2.0 ** -13


@pytest.mark.parametrize("q_type,dtype", [(F32, I8), (F32, E4M3), (F16, I8), (BF16, E4M3)])
@pytest.mark.parametrize("heads,kv_heads,dim,tokens", [(8, 2, 64, 512), (16, 1, 128, 8), (24, 1, 256, 3000)])
def test_scales_far_apart(q_type, dtype, heads, kv_heads, dim, tokens):
    """Scales of V from 2^-20 to 2^20, and tokens whose scale is 10^8 times as large without any weight: what the
    others add up to keeps its bits."""
    batch = 6
    shape = (batch, -(-tokens // 8) * 8, kv_heads, dim)
    k, v = codes(shape, dtype), codes(shape, dtype)
    ks = torch.full(shape[:3], 0.01, device=DEV)
    vs = 0.01 * torch.exp2(torch.rand(shape[:3], device=DEV) * 40 - 20)
    vs[0] = vs[1] = 0.01
    q = torch.randn((batch, heads, dim), device=DEV).to(q_type)
    # first, last or in the middle: a key so far on the other side of every query that its weight is 0
    q[:, :, 0] = 16
    for b, at in ((0, 0), (1, tokens - 1), (2, tokens // 2), (3, 0)):
        k[b, at] = 0
        k[b, at, :, 0] = torch.tensor(-100.0).to(dtype)
        ks[b, at], vs[b, at] = 10, 1e6
    n = torch.full((batch,), tokens, device=DEV, dtype=torch.int32)
    out, (want, d) = attend(q, k, v, n, ks, vs), exact(q, k, v, n, ks, vs)
    check(out, want, d)
    if q_type is F32:  # errors of either sign
        assert float(((out - want).norm(dim=(1, 2)) / want.norm(dim=(1, 2))).max()) <= 1e-5


@pytest.mark.parametrize("q_type,dtype", [(F32, I8), (BF16, E4M3)])
def test_scales_while_scores_grow(q_type, dtype):
    """Scores that rise tile by tile, and V's scales that fall or rise with them, far enough for each to be out
    of the other's range at the end; tokens without scale; all scales 0."""
    batch, tokens, dim = 5, 640, 64
    shape = (batch, tokens, 2, dim)
    k, v = codes(shape, dtype), codes(shape, dtype)
    t = torch.linspace(0, 1, tokens, device=DEV)[None, :, None].expand(shape[:3])
    k[..., 0] = torch.tensor(64.0).to(dtype)
    ks = 0.1 * t
    vs = torch.stack([torch.exp2(-60 * t[0]), torch.exp2(60 * t[1] - 60), torch.exp2(-60 * t[2]) * (t[2] > 0.5),
                      torch.zeros_like(t[3]), torch.exp2(40 * torch.rand(t[4].shape, device=DEV) - 20)])
    q = torch.randn((batch, 8, dim), device=DEV).to(q_type)
    q[:, :, 0] = 30
    n = torch.full((batch,), tokens, device=DEV, dtype=torch.int32)
    out = attend(q, k, v, n, ks, vs)
    assert not out[3].any()
    # of a score, the largest term is 30 * 6.4 and the others are small: their sum's error is that of the largest
    check(out, *exact(q, k, v, n, ks, vs))


@pytest.mark.parametrize("q_type,dtype", [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("dim", [64, 80, 36])
def test_infinite_keys(q_type, dtype, dim):
    """A key that makes a score -inf has no weight, whatever pieces the product is made of; a sequence of
    such keys alone gets zeros, and a score of +inf NaN."""
    k, v = (torch.randn((4, 24, 2, dim), device=DEV).to(dtype) for _ in range(2))
    q = torch.randn((4, 8, dim), device=DEV).to(q_type)
    q[:, :, 3] = 1.7
    n = torch.tensor([20, 7, 17, 20], device=DEV, dtype=torch.int32)
    k[0, 19, :, 3] = k[1, 6, :, 3] = -torch.inf
    k[2, :, :, 3] = -torch.inf
    k[3, 5, :, 3] = torch.inf
    out = attend(q, k, v, n)
    check(out[:2], *exact(q[:2], k[:2], v[:2], n[:2] - 1))
    assert not out[2].any() and bool(out[3].isnan().all())


@pytest.mark.parametrize("q_type,dtype,batch,heads,dim", [(F16, F16, 1, 4, 256), (F32, BF16, 2, 16, 128), (BF16, I8, 40, 8, 64),
                                                          (F32, F32, 1, 1, 32)])
def test_long_joins_repeat(q_type, dtype, batch, heads, dim):
    """Sequences in many parts, joined by all teams of a block: the same bits every time, and right."""
    tokens = 30000 // batch // 8 * 8
    scaled = dtype is I8
    k, v = (codes((batch, tokens, 1, dim), dtype) if scaled else torch.randn((batch, tokens, 1, dim), device=DEV).to(dtype)
            for _ in range(2))
    z = [0.01 * torch.rand((batch, tokens, 1), device=DEV) if scaled else None for _ in range(2)]
    q = torch.randn((batch, heads, dim), device=DEV).to(q_type)
    n = torch.randint(tokens // 2, tokens + 1, (batch,), device=DEV, dtype=torch.int32)
    out = attend(q, k, v, n, *z)
    check(out, *exact(q, k, v, n, *z))
    for _ in range(50):
        assert torch.equal(attend(q, k, v, n, *z), out)


@pytest.mark.parametrize("q_type,dtype", [(F16, F16), (BF16, BF16), (F16, I8), (BF16, E4M3), (F32, I8), (F32, F32)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (32, 2, 128), (16, 1, 256), (24, 2, 80), (3, 1, 32)])
def test_long_lines_whose_scores_grow_late(q_type, dtype, heads, kv_heads, dim):
    """Hundreds of tiles a warp, then scores higher by 6 and scales of V 1000 times as large, by values of the other
    sign: what was added up before has to be scaled down. The first 256 of 512 tokens are seen 400 times each, so the
    two halves weigh about the same. Sums are off by 2^-14 A at most (as above, and scores of up to 12 by 2^-20 each), pieces
    of bf16 by 2^-16 A."""
    batch, times = 32, 400
    scaled = dtype in (I8, E4M3)
    k = (torch.randn((1, 512, kv_heads, dim), device=DEV) * 1.5).round().clamp(-4, 4)
    k[:, 256:, :, 0] = 64
    k[:, :256, :, 0] = 0
    v = torch.randn((1, 512, kv_heads, dim), device=DEV).mul(4).round().clamp(-12, 12) + 40
    v[:, 256:] *= -1
    z = [torch.full((1, 512, kv_heads), x, device=DEV) for x in (0.25, 0.01)]
    z[1][:, 256:] = 10
    if not scaled:
        k, v = k * z[0][..., None], v * z[1][..., None]
        z = [None, None]
    k, v = k.to(dtype), v.to(dtype)
    q = torch.randn((batch, heads, dim), device=DEV) * 0.25
    q[:, :, 0] = 6 / 16 * dim ** 0.5
    q = q.to(q_type)
    pages = [None if x is None else x.unflatten(1, (-1, 8)).flatten(0, 1) for x in (k, v, *z)]
    order = torch.cat([torch.arange(32).repeat(times), torch.arange(32, 64)]).to(DEV, torch.int32)
    n = torch.full((batch,), len(order) * 8, device=DEV, dtype=torch.int32)
    got = paged_attention(q, *pages[:2], order.expand(batch, -1), n, k_scale=pages[2], v_scale=pages[3])
    values = [x.double() if y is None else x.double() * y.double()[..., None] for x, y in ((k, z[0]), (v, z[1]))]
    s = torch.einsum("bhgd,thd->bhgt", q.double().unflatten(1, (kv_heads, -1)), values[0][0]) * dim ** -0.5
    s[..., :256] += torch.tensor(float(times)).double().log()
    p = torch.softmax(s, -1)
    o, A = (torch.einsum("bhgt,thd->bhgd", p, x).flatten(1, 2) for x in (values[1][0], values[1][0].abs()))
    check(got, o, A * (2.0 ** -14 + (2.0 ** -16 if dtype is BF16 else 0)))
