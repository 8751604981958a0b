"""The paged key-value cache's operators on device arrays, against plain 64-bit forms
(``paged_reference``): writes and reads bit for bit, attention within derived bounds."""

from __future__ import annotations

import math

import pytest
import torch

from metellus_b200 import cache_read, cache_write, paged_attention
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16, I8, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn
DEV = "cuda"


@pytest.fixture(autouse=True)
def _device(cuda_device):
    torch.manual_seed(5)


def raw(x):
    """8-bit floats as bytes, for comparison and indexing."""
    return x.view(torch.uint8) if x.dtype is E4M3 else x


def new_cache(pages, ps, heads, dim, dtype, order="nhd", fill=True):
    """(k, v, k_scale, v_scale); ``order`` is the order of (tokens, heads) in memory."""
    def one():
        shape = (pages, ps, heads, dim) if order == "nhd" else (pages, heads, ps, dim)
        x = torch.randn(shape, device=DEV)
        x = (x * (40 if dtype is I8 else 100 if dtype is E4M3 else 1)).clamp(-440, 440)
        x = x.round().clamp(-127, 127).to(I8) if dtype is I8 else x.to(dtype)
        return x if order == "nhd" else x.transpose(1, 2)

    def scales():
        shape = (pages, ps, heads) if order == "nhd" else (pages, heads, ps)
        z = 0.002 + 0.03 * torch.rand(shape, device=DEV)
        return z if order == "nhd" else z.transpose(1, 2)

    z = (scales(), scales()) if dtype in (I8, E4M3) else (None, None)
    return (one(), one()) + z


def kw(c):
    return {"k_scale": c[2], "v_scale": c[3]}


# -- writing and reading ------------------------------------------------------------------


@pytest.mark.parametrize("x_type", [F32, F16, BF16])
@pytest.mark.parametrize("dtype", [F32, F16, BF16, I8, E4M3])
@pytest.mark.parametrize("n,ps,heads,dim,order", [
    (1, 16, 8, 128, "nhd"), (77, 16, 8, 128, "nhd"), (50, 1, 1, 1, "nhd"), (33, 24, 3, 7, "nhd"),
    (40, 8, 2, 80, "hnd"), (130, 32, 5, 64, "hnd"), (19, 64, 1, 256, "nhd"), (21, 16, 2, 36, "nhd")])
def test_write_and_read(x_type, dtype, n, ps, heads, dim, order):
    pages = -(-n // ps) + 3
    c = new_cache(pages, ps, heads, dim, dtype, order)
    before = [None if x is None else x.clone() for x in c]
    # every second tensor wider than its rows: strides that are not the packed ones
    wide = torch.randn((n, 2 * heads, dim + 8), device=DEV).to(x_type)
    k, v = wide[:, :heads, :dim], wide[:, heads:, 8:]
    slots = torch.randperm(pages * ps, device=DEV)[:n]
    slots[n // 2:n // 2 + 1] = -1
    if n > 10:
        slots[3], slots[4] = pages * ps, 2 ** 40
    at = slots if n % 2 else slots.clamp(max=2 ** 31 - 1).int()
    cache_write(k, v, c[0], c[1], at, **kw(c))
    keep = (slots >= 0) & (slots < pages * ps)
    page, off = slots[keep] // ps, slots[keep] % ps
    for x, cache, scale, old, old_scale in ((k, c[0], c[2], before[0], before[2]), (v, c[1], c[3], before[1], before[3])):
        want = old.float() if dtype is E4M3 else old.clone()
        if scale is None:
            want[page, off] = x[keep].to(dtype)
        else:
            code, z = ref.codes(x[keep], dtype)
            want[page, off] = code.to(want.dtype)
            want_scale = old_scale.clone()
            want_scale[page, off] = z
            assert torch.equal(scale, want_scale)
        # the rows written and every other one, bit for bit
        assert torch.equal(raw(cache), raw(want.to(dtype)))
    for out_type in (F32, F16, BF16):
        got = cache_read(c[0], c[1], at, dtype=out_type, **kw(c))
        for y, cache, scale in ((got[0], c[0], c[2]), (got[1], c[1], c[3])):
            want = torch.zeros((n, heads, dim), device=DEV)
            rows = cache.float()
            want[keep] = (rows if scale is None else rows * scale[..., None])[page, off]
            assert y.dtype is out_type and torch.equal(y, want.to(out_type))


@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("x_type", [F32, F16, BF16])
def test_codes_at_borders(dtype, x_type):
    """Quotients that are ties or next to one, zeros, tiny and huge rows, rows with
    infinities and NaN."""
    top = ref.CODE_MAX[dtype]
    rows = torch.zeros((1200, 1, 128), device=DEV)
    for i in range(1000):
        s = torch.rand((), device=DEV) * 10.0 ** (i % 7 - 3)
        half = torch.randint(0, 127, (127,), device=DEV) + 0.5
        if dtype is E4M3:
            half = half * torch.exp2(torch.randint(-9, 3, (127,), device=DEV).float())
        rows[i, 0, :127] = half * s * torch.where(torch.rand(127, device=DEV) < 0.5, 1.0, 1.0 + 6e-8)
        rows[i, 0, 127] = top * s
    rows[1000] = 0
    rows[1001, 0, 5] = math.inf
    rows[1002, 0, 5] = math.nan
    rows[1003, 0, 5] = -math.inf
    rows[1004] = 1e-30
    rows[1005] = torch.randn(128, device=DEV) * 3e38 / 10
    x = rows.clamp(-6e4, 6e4).where(torch.isfinite(rows), rows).to(x_type) if x_type is F16 else rows.to(x_type)
    c = new_cache(75, 16, 1, 128, dtype)
    slots = torch.arange(1200, device=DEV)
    cache_write(x, -x, c[0], c[1], slots, **kw(c))
    for y, cache, scale in ((x, c[0], c[2]), (-x, c[1], c[3])):
        code, z = ref.codes(y, dtype)
        assert torch.equal(scale.flatten(0, 1).nan_to_num(-7), z.nan_to_num(-7))
        assert torch.equal(cache.float().flatten(0, 1), code.float())
    k, _ = cache_read(c[0], c[1], slots, **kw(c))
    assert bool(torch.isnan(k[1001:1004]).all()) and bool(torch.isfinite(k[:1000]).all()) and not k[1000].any()


@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("dim", [64, 36])
def test_codes_of_smallest_rows(dtype, dim):
    """Scales around and below fp32's smallest normal number, down to a few of its steps,
    where largest / scale passes the largest code by up to half."""
    x = torch.randn((400, 1, dim), device=DEV) * torch.exp2(-torch.linspace(90, 149, 400, device=DEV))[:, None, None]
    x[::7, 0, 0] = -0.0
    c = new_cache(25, 16, 1, dim, dtype)
    cache_write(x, -x, c[0], c[1], torch.arange(400, device=DEV), **kw(c))
    for y, cache, scale in ((x, c[0], c[2]), (-x, c[1], c[3])):
        code, z = ref.codes(y, dtype)
        assert torch.equal(scale.flatten(0, 1), z)
        assert torch.equal(cache.float().flatten(0, 1), code.float().clamp(-ref.CODE_MAX[dtype], ref.CODE_MAX[dtype]))


def test_read_into_strided_rows():
    """Heads first, as the batched attention of programs takes K."""
    c = new_cache(9, 16, 4, 64, I8)
    slots = torch.randperm(144, device=DEV)[:100]
    guard = torch.full((6, 104, 64), 7.0, device=DEV)
    other = torch.full((4, 100, 64), 7.0, device=DEV)
    k, v = cache_read(c[0], c[1], slots, out=(guard[1:5, 2:102].transpose(0, 1), other.transpose(0, 1)), **kw(c))
    want = cache_read(c[0], c[1], slots, **kw(c))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    outside = guard.clone()
    outside[1:5, 2:102] = 7.0
    assert bool((outside == 7.0).all())


def test_repeated_slot_leaves_the_others():
    c = new_cache(4, 16, 2, 64, BF16)
    x = torch.randn((20, 2, 64), device=DEV).bfloat16()
    slots = torch.arange(20, device=DEV)
    slots[7] = slots[3]
    cache_write(x, x, c[0], c[1], slots)
    rows = c[0].flatten(0, 1)
    keep = [i for i in range(20) if i not in (3, 7)]
    assert torch.equal(rows[keep], x[keep])


# -- attention ----------------------------------------------------------------------------


def make(lengths, heads, kv_heads, dim, ps, q_type, dtype, order="nhd", spare=4, extra_width=2):
    used = [-(-n // ps) for n in lengths]
    pages = sum(used) + spare
    c = new_cache(pages, ps, kv_heads, dim, dtype, order)
    order_ = torch.randperm(pages, dtype=torch.int32)
    tables = torch.full((len(lengths), max(used, default=0) + extra_width), -1, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        tables[b, :u] = order_[at:at + u]
        at += u
    q = (torch.randn((len(lengths), heads, dim), device=DEV) * 2).to(q_type)
    return q, c, tables.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)


def compare(q, c, tables, lengths, **more):
    out, lse = paged_attention(q, c[0], c[1], tables, lengths, return_lse=True, **kw(c), **more)
    want, want_lse, tol, lse_tol = ref.attention(q, c[0], c[1], tables, lengths, **kw(c), **more)
    assert out.dtype is q.dtype
    ref.check(out, want, tol, "out")
    ref.check(lse, want_lse, lse_tol, "lse")
    ok = torch.isfinite(want)
    if q.dtype is F32 and bool(ok.any()) and float(want[ok].norm()) > 0:
        assert float((out.double() - want)[ok].norm() / want[ok].norm()) <= 1e-5
    return out, lse


PAIRS = [(F32, F32), (F16, F16), (F32, F16), (BF16, BF16), (F32, BF16), (F32, I8), (F16, I8), (BF16, I8),
         (F32, E4M3), (F16, E4M3), (BF16, E4M3)]


@pytest.mark.parametrize("q_type,dtype", PAIRS)
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,ps", [
    ([1], 8, 8, 128, 16), ([100], 32, 8, 128, 16), ([0, 1, 15, 16, 17, 63, 64, 65, 1000], 8, 2, 64, 16),
    ([257, 3, 0, 129], 5, 1, 128, 24), ([5000], 4, 1, 128, 8), ([333, 334], 16, 1, 256, 1), ([70, 700], 24, 1, 64, 64),
    ([40, 90], 6, 3, 80, 16), ([31, 200], 3, 3, 96, 32), ([77], 33, 1, 32, 128)])
def test_attention(q_type, dtype, lengths, heads, kv_heads, dim, ps):
    compare(*make(lengths, heads, kv_heads, dim, ps, q_type, dtype))


@pytest.mark.parametrize("q_type,dtype", [(F32, F32), (BF16, BF16), (BF16, I8), (F16, F16)])
@pytest.mark.parametrize("batch,longest,extra_width", [(300, 400, 2), (700, 40, 0), (700, 40, 900), (1, 40000, 0), (1, 300, 5000),
                                                       (2, 70, 20)])
def test_attention_batches(q_type, dtype, batch, longest, extra_width):
    """More sequences than threads, more items than blocks, fewer units than blocks."""
    lengths = torch.randint(0, longest + 1, (batch,)).tolist()
    lengths[0] = longest
    compare(*make(lengths, 6, 3, 64, 16, q_type, dtype, extra_width=extra_width))


@pytest.mark.parametrize("q_type,dtype", [(F32, F32), (BF16, BF16), (F16, F16), (F32, I8), (BF16, E4M3)])
@pytest.mark.parametrize("heads,dim", [(8, 128), (6, 64), (16, 256), (6, 36)])
def test_attention_padded_batch(q_type, dtype, heads, dim):
    """Sequences without tokens alone and in runs, first and last, between long and short ones:
    their rows are zeros, written over what was there."""
    lengths = [0, 0, 700, 0, 3, 0, 0, 0, 40, 1, 0, 1500] + [0] * 70 + [17, 0, 90] + [0] * 40
    q, c, tables, n = make(lengths, heads, 2, dim, 16, q_type, dtype)
    out = torch.full_like(q, math.nan)
    paged_attention(q, c[0], c[1], tables, n, out=out, **kw(c))
    assert not out[n == 0].any()
    assert torch.equal(out, compare(q, c, tables, n)[0])


@pytest.mark.parametrize("q_type,dtype", PAIRS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(11, 1, 64), (32, 2, 96), (40, 2, 128), (33, 1, 32), (16, 1, 256), (20, 1, 192)])
def test_attention_wide_groups(q_type, dtype, heads, kv_heads, dim):
    """Tables wide enough for many tiles a warp: 16 query heads are taken at a time."""
    compare(*make([0, 5, 300, 2500, 1], heads, kv_heads, dim, 128, q_type, dtype, extra_width=4000))


@pytest.mark.parametrize("q_type,dtype", [(F32, F32), (BF16, BF16), (F32, I8), (F16, E4M3)])
@pytest.mark.parametrize("dim", [1, 7, 36, 100, 200, 250])
def test_attention_odd_head_dims(q_type, dtype, dim):
    compare(*make([0, 50, 300], 6, 2, dim, 16, q_type, dtype))


@pytest.mark.parametrize("q_type,dtype", PAIRS)
@pytest.mark.parametrize("dim", [4, 8, 16, 24, 32, 48])
def test_attention_small_head_dims(q_type, dtype, dim):
    compare(*make([0, 1, 50, 300, 2000], 12, 3, dim, 16, q_type, dtype))


@pytest.mark.parametrize("q_type,dtype", [(F32, F32), (BF16, BF16), (F32, F16), (BF16, I8), (F32, E4M3)])
@pytest.mark.parametrize("window", [1, 16, 100, 5000])
def test_attention_window(q_type, dtype, window):
    compare(*make([0, 5, 100, 101, 1000, 3000], 8, 2, 128, 16, q_type, dtype), window=window)


@pytest.mark.parametrize("q_type,dtype", [(F32, F32), (BF16, BF16), (F16, F16), (F32, I8), (BF16, E4M3)])
def test_attention_strides(q_type, dtype):
    """Heads before tokens in the cache's memory, q and out inside wider tensors, a table
    and lengths that are slices."""
    q, c, tables, lengths = make([0, 50, 301, 7], 8, 4, 64, 16, q_type, dtype, order="hnd")
    wide = torch.zeros((4, 24, 96), device=DEV, dtype=q_type)
    wide[:, 8:16, 32:] = q
    more = torch.full((4, tables.shape[1] + 5), 10 ** 9, device=DEV, dtype=torch.int32)
    more[:, 2:2 + tables.shape[1]] = tables
    pairs = torch.zeros((4, 2), device=DEV, dtype=torch.int32)
    pairs[:, 1] = lengths
    out = torch.full((4, 10, 70), 9.0, device=DEV, dtype=q_type)
    got = paged_attention(wide[:, 8:16, 32:], c[0], c[1], more[:, 2:2 + tables.shape[1]], pairs[:, 1],
                          out=out[:, 1:9, 3:67], **kw(c))
    want, _, tol, _ = ref.attention(q, c[0], c[1], tables, lengths, **kw(c))
    ref.check(got, want, tol)
    out[:, 1:9, 3:67] = 9.0
    assert bool((out == 9.0).all())


@pytest.mark.parametrize("q_type,dtype", [(F32, F32), (BF16, BF16), (F16, F16), (F32, I8), (BF16, E4M3)])
def test_attention_ignores_what_is_not_visible(q_type, dtype):
    """NaN and infinities in unused slots, in other pages and behind the window, lengths
    behind the table's end or negative, page numbers outside the cache."""
    q, c, tables, lengths = make([0, 50, 301, 7, 130], 8, 2, 128, 16, q_type, dtype)
    seen = torch.zeros(c[0].shape[:2], dtype=torch.bool, device=DEV)
    n, window = lengths.tolist(), 90
    for b in range(len(n)):
        t = torch.arange(max(0, n[b] - window), n[b], device=DEV)
        seen[tables[b].long()[t // 16], t % 16] = True
    bad = math.nan
    for x in c:
        if x is None:
            continue
        if x.dtype is I8:
            x[~seen] = 127
        elif x.dtype is E4M3:
            x.view(torch.uint8)[~seen] = 0x7F
        else:
            x[~seen] = bad
            x[-1][~seen[-1]] = math.inf
    compare(q, c, tables, lengths, window=window)
    # a hole in the middle of a sequence, a length over the table's width, one below zero
    tables[2, 17], tables[4, 5] = -5, c[0].shape[0]
    lengths[1], lengths[0] = 10 ** 6, -3
    tables[1, 4:] = -1
    compare(q, c, tables, lengths, window=0 if dtype is F32 else 90)


@pytest.mark.parametrize("q_type,dtype", [(F32, F32), (BF16, BF16), (F16, I8)])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 0.02, 0.5])
def test_attention_scale(q_type, dtype, scale):
    compare(*make([0, 1, 77, 400], 8, 2, 64, 16, q_type, dtype), scale=scale)


@pytest.mark.parametrize("q_type,dtype", [(F32, F32), (BF16, BF16), (F32, I8)])
def test_attention_large_scores(q_type, dtype):
    """A row that attends to one token alone, and scores far apart in magnitude."""
    q, c, tables, lengths = make([100, 2000], 4, 1, 64, 16, q_type, dtype)
    q *= 60
    out, _ = paged_attention(q, c[0], c[1], tables, lengths, return_lse=True, **kw(c))
    want, _, tol, _ = ref.attention(q, c[0], c[1], tables, lengths, **kw(c))
    ref.check(out, want, tol)
    q *= 0
    compare(q, c, tables, lengths)


@pytest.mark.parametrize("q_type,dtype,dim", [(BF16, BF16, 128), (F32, I8, 128), (F32, F32, 64), (BF16, BF16, 36), (F16, E4M3, 80)])
def test_caches_of_over_32_bits(q_type, dtype, dim):
    """Pages behind 2^31 elements (and 2^32 bytes) of a cache: the same, bit for bit, as in a small one."""
    q, c, tables, n = make([5, 700, 90], 8, 2, dim, 16, q_type, dtype, spare=0)
    used = c[0].shape[0]
    pages = (2 ** 31 + 2 ** 30 * (4 // dtype.itemsize)) // (16 * 2 * dim) + used
    big = [None if x is None else torch.empty((pages, *x.shape[1:]), device=DEV, dtype=x.dtype) for x in c]
    slots = torch.arange(used * 16, device=DEV) + (pages - used) * 16
    for x, y in zip(big, c):
        if x is not None:
            raw(x)[pages - used:] = raw(y)
    far = torch.where(tables >= 0, tables + (pages - used), tables)
    assert torch.equal(paged_attention(q, big[0], big[1], far, n, **kw(big)), paged_attention(q, c[0], c[1], tables, n, **kw(c)))
    rows = cache_read(big[0], big[1], slots, **kw(big))
    here = cache_read(c[0], c[1], slots - slots[0], **kw(c))
    assert torch.equal(rows[0], here[0]) and torch.equal(rows[1], here[1])
    x = torch.randn((used * 16, 2, dim), device=DEV)
    cache_write(x, -x, big[0], big[1], slots, **kw(big))
    cache_write(x, -x, c[0], c[1], slots - slots[0], **kw(c))
    for y, z in zip(big, c):
        assert z is None or torch.equal(raw(y)[pages - used:], raw(z))


def test_nothing_to_do():
    c = new_cache(3, 16, 2, 64, BF16)
    q = torch.zeros((0, 4, 64), device=DEV, dtype=BF16)
    i = lambda *s: torch.zeros(s, device=DEV, dtype=torch.int32)  # noqa: E731
    assert paged_attention(q, c[0], c[1], i(0, 5), i(0)).shape == (0, 4, 64)
    q = torch.ones((2, 4, 64), device=DEV, dtype=BF16)
    out, lse = paged_attention(q, c[0], c[1], i(2, 0), i(2) + 9, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    empty = [x[:0] for x in c[:2]]
    out, lse = paged_attention(q, empty[0], empty[1], i(2, 3), i(2) + 9, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    rows = torch.ones((3, 2, 64), device=DEV, dtype=BF16)
    cache_write(rows, rows, empty[0], empty[1], i(3))
    cache_write(rows[:0], rows[:0], c[0], c[1], i(0))
    assert not cache_read(empty[0], empty[1], i(3))[0].any()
    assert cache_read(c[0], c[1], i(0))[0].shape == (0, 2, 64)


# -- together, and as programs call them -----------------------------------------------------


@pytest.mark.parametrize("x_type,dtype,tol", [(F32, F32, 1e-5), (F32, BF16, 1e-2), (BF16, I8, 3e-2), (F32, E4M3, 8e-2)])
def test_decoding_step_by_step(x_type, dtype, tol):
    """Prompts written at once, then one token a step: every step's attention against
    attention over the rows as they came. The tolerance is the caches' rounding: a step of
    2^-8 (bf16), 1 / 127 / 2 of the row's largest, 2^-4, which softmax averages."""
    heads, hk, dim, ps, steps = 8, 2, 64, 16, 20
    prompt = [13, 32, 1]
    width = (max(prompt) + steps) // ps + 1
    tables = torch.randperm(3 * width, device=DEV, dtype=torch.int32).view(3, width)
    c = new_cache(3 * width, ps, hk, dim, dtype)
    keys = [torch.randn((n, hk, dim), device=DEV).to(x_type) for n in prompt]
    vals = [torch.randn((n, hk, dim), device=DEV).to(x_type) for n in prompt]

    def slots_of(b, t):
        return tables[b].long()[t // ps] * ps + t % ps

    cache_write(torch.cat(keys), torch.cat(vals), c[0], c[1],
                torch.cat([slots_of(b, torch.arange(n, device=DEV)) for b, n in enumerate(prompt)]), **kw(c))
    lengths = torch.tensor(prompt, device=DEV, dtype=torch.int32)
    for _ in range(steps):
        k, v = (torch.randn((3, hk, dim), device=DEV).to(x_type) for _ in range(2))
        q = torch.randn((3, heads, dim), device=DEV).to(x_type)
        cache_write(k, v, c[0], c[1], torch.stack([slots_of(b, lengths[b].long()) for b in range(3)]), **kw(c))
        lengths += 1
        out = paged_attention(q, c[0], c[1], tables, lengths, **kw(c))
        for b in range(3):
            keys[b], vals[b] = torch.cat([keys[b], k[b:b + 1]]), torch.cat([vals[b], v[b:b + 1]])
            s = torch.einsum("hgd,thd->hgt", q[b].double().view(hk, heads // hk, dim), keys[b].double()) * dim ** -0.5
            want = torch.einsum("hgt,thd->hgd", torch.softmax(s, -1), vals[b].double()).flatten(0, 1)
            assert float((out[b].double() - want).norm() / want.norm()) <= tol
    assert [len(x) for x in keys] == lengths.tolist()


def test_captured_steps_share_nothing():
    """Two graphs captured from the same call sites, replayed one after the other and at
    once on two streams, with new lengths and tables between replays."""
    cases = []
    for seed in range(2):
        torch.manual_seed(seed)
        q, c, tables, lengths = make([3000, 500, 40], 8, 2, 128, 16, BF16, BF16)
        paged_attention(q, c[0], c[1], tables, lengths)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=stream):
            new = q[:, :2, :] * 2
            cache_write(new, new, c[0], c[1], lengths - 1)
            out = paged_attention(q, c[0], c[1], tables, lengths)
        cases.append((q, c, tables, lengths, graph, out, stream))
    torch.cuda.synchronize()
    for turn in range(4):
        for q, c, tables, lengths, graph, out, stream in cases:
            lengths -= 7
            q.copy_(torch.randn_like(q))
        torch.cuda.synchronize()
        for q, c, tables, lengths, graph, out, stream in cases:
            with torch.cuda.stream(stream if turn % 2 else torch.cuda.current_stream()):
                graph.replay()
        torch.cuda.synchronize()
        for q, c, tables, lengths, graph, out, stream in cases:
            want, _, tol, _ = ref.attention(q, c[0], c[1], tables, lengths)
            ref.check(out, want, tol)


@pytest.mark.parametrize("longest,extra_width", [(16, 4000), (3000, 0)])
def test_calls_follow_one_another(longest, extra_width):
    """What comes after an attention (here a write into the pages that it reads) waits for all of
    it: with no sequence to join, though the tables are wide, and with long ones."""
    lengths = torch.randint(1, longest + 1, (64,)).tolist()
    q, c, tables, n = make(lengths, 32, 8, 128, 16, BF16, BF16, extra_width=extra_width)
    want = paged_attention(q, c[0], c[1], tables, n)
    slots = torch.arange(c[0].shape[0] * 16, device=DEV)
    kept = cache_read(c[0], c[1], slots)
    other = [torch.full_like(x, 9.0) for x in kept]
    for _ in range(20):
        out = paged_attention(q, c[0], c[1], tables, n)
        cache_write(*other, c[0], c[1], slots)
        cache_write(*kept, c[0], c[1], slots)
        again = paged_attention(q, c[0], c[1], tables, n)
        assert torch.equal(out, want) and torch.equal(again, want)


def test_runs_on_the_current_stream():
    """Work queued before a call on the current stream is seen by it, on a side stream and on
    the default one; results are the same in repeated calls."""
    q, c, tables, lengths = make([4000, 100], 8, 2, 128, 16, BF16, E4M3)
    want = paged_attention(q, c[0], c[1], tables, lengths, **kw(c)).clone()
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            late = torch.zeros_like(q)
            torch.cuda._sleep(20_000_000)
            late.copy_(q)
            got = paged_attention(late, c[0], c[1], tables, lengths, **kw(c))
            rows = cache_read(c[0], c[1], torch.arange(5, device=DEV), **kw(c))
        stream.synchronize()
        assert torch.equal(got, want)
        assert torch.equal(rows[0], c[0].float().flatten(0, 1)[:5] * c[2].flatten(0, 1)[:5, :, None])


# -- refusals ------------------------------------------------------------------------------


def test_refusals_leave_everything_alone():
    q, c, tables, lengths = make([20, 30], 8, 2, 64, 16, BF16, BF16)
    k = torch.randn((2, 2, 64), device=DEV).bfloat16()
    slots = torch.tensor([1, 2], device=DEV)
    before = c[0].clone()
    i8 = new_cache(4, 16, 2, 64, I8)
    for error, call in [
        (ValueError, lambda: paged_attention(q.half(), c[0], c[1], tables, lengths)),
        (ValueError, lambda: paged_attention(q[:, :7], c[0], c[1], tables, lengths)),
        (ValueError, lambda: paged_attention(q[..., :32], c[0], c[1], tables, lengths)),
        (ValueError, lambda: paged_attention(q, c[0], c[1], tables.long(), lengths)),
        (ValueError, lambda: paged_attention(q, c[0], c[1], tables, lengths.long())),
        (ValueError, lambda: paged_attention(q, c[0], c[1], tables[:1], lengths)),
        (ValueError, lambda: paged_attention(q, c[0], c[1], tables, lengths[:1])),
        (ValueError, lambda: paged_attention(q, c[0], c[1].half(), tables, lengths)),
        (ValueError, lambda: paged_attention(q, i8[0], i8[1], tables, lengths)),
        (ValueError, lambda: paged_attention(q, c[0], c[1], tables, lengths, k_scale=i8[2], v_scale=i8[3])),
        (ValueError, lambda: paged_attention(q, c[0], c[1], tables, lengths, scale=math.inf)),
        (ValueError, lambda: paged_attention(q, c[0], c[1], tables, lengths, window=-1)),
        (ValueError, lambda: paged_attention(q, c[0], c[1], tables, lengths, out=torch.zeros_like(q).float())),
        (ValueError, lambda: paged_attention(q, c[0], c[1], tables, lengths, out=q[:, :1].expand(-1, 8, -1))),
        (ValueError, lambda: paged_attention(q, c[0].cpu(), c[1], tables, lengths)),
        (ValueError, lambda: paged_attention(q.transpose(1, 2).contiguous().transpose(1, 2), c[0], c[1], tables, lengths)),
        (TypeError, lambda: paged_attention(q, c[0], c[1], tables.tolist(), lengths)),
        (ValueError, lambda: paged_attention(q.detach().requires_grad_(), c[0], c[1], tables, lengths)),
        (ValueError, lambda: cache_write(k, k[:1], c[0], c[1], slots)),
        (ValueError, lambda: cache_write(k, k.float(), c[0], c[1], slots)),
        (ValueError, lambda: cache_write(k[..., :32], k[..., :32], c[0], c[1], slots)),
        (ValueError, lambda: cache_write(k, k, c[0], c[1], slots.float())),
        (ValueError, lambda: cache_write(k, k, c[0][:1].expand(5, -1, -1, -1), c[1][:5], slots)),
        (ValueError, lambda: cache_write(k, k, i8[0], i8[1], slots, k_scale=i8[2])),
        (ValueError, lambda: cache_write(k, k, i8[0], i8[1], slots, k_scale=i8[2], v_scale=i8[3][:2])),
        (ValueError, lambda: cache_read(c[0], c[1], slots, dtype=torch.float64)),
        (ValueError, lambda: cache_read(c[0], c[1], slots, out=(k[:1], k))),
    ]:
        with pytest.raises(error):
            call()
    torch.cuda.synchronize()
    assert torch.equal(c[0], before)
