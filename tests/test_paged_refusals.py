"""Argument checks of the paged cache's C entry points, on the CPU: nothing here can reach
a launch (the pointers are numbers, and every call has something that does not fit)."""

from __future__ import annotations

import ctypes

import pytest

from metellus_b200.runtime import backend
from metellus_b200.runtime.backend import ARRAY_DTYPES, MtArray, MtPagedCache


def array(dtype, shape, strides=None, ptr=4096):
    if strides is None:
        strides, step = [], 1
        for n in reversed(shape):
            strides.insert(0, step)
            step *= n
    return MtArray(ptr, ARRAY_DTYPES[dtype], len(shape), tuple(shape), tuple(strides))


def cache(dtype="bfloat16", pages=4, page_size=16, heads=2, dim=64, **other):
    c = MtPagedCache(array(dtype, (pages, page_size, heads, dim)), array(dtype, (pages, page_size, heads, dim)))
    if dtype in ("int8", "float8_e4m3fn"):
        c.k_scale = array("float32", (pages, page_size, heads))
        c.v_scale = array("float32", (pages, page_size, heads))
    for name, x in other.items():
        setattr(c, name, x)
    return c


def refused(rc, match):
    assert rc == 2
    with pytest.raises(ValueError, match=match):
        backend._check(rc)


def attend(match, **other):
    a = dict(q=array("bfloat16", (3, 4, 64)), cache=cache(), tables=array("int32", (3, 5)),
             lengths=array("int32", (3,)), out=array("bfloat16", (3, 4, 64)), lse=None, scale=0.125, window=0)
    a.update(other)
    refused(backend.lib().mt_paged_attention(0, a["q"], a["cache"], a["tables"], a["lengths"], a["out"], a["lse"],
                                             a["scale"], a["window"], None, 0, None), match)


@pytest.mark.parametrize("match,other", [
    ("q must have 3 dimensions", {"q": array("bfloat16", (3, 64))}),
    ("q cannot be int8", {"q": array("int8", (3, 4, 64))}),
    ("q is missing", {"q": None}),
    ("head_dim 32, the cache 64", {"q": array("bfloat16", (3, 4, 32))}),
    ("5 query heads are not a multiple of 2", {"q": array("bfloat16", (3, 5, 64))}),
    ("does not go with a cache of bfloat16", {"q": array("float16", (3, 4, 64))}),
    ("does not go with a cache of float32", {"cache": cache("float32")}),
    ("last dimension of q must be contiguous", {"q": array("bfloat16", (3, 4, 64), (256, 1, 4))}),
    ("q has no memory", {"q": array("bfloat16", (3, 4, 64), ptr=0)}),
    ("not aligned to its elements", {"q": array("bfloat16", (3, 4, 64), ptr=4097)}),
    ("negative stride", {"q": array("bfloat16", (3, 4, 64), (-256, 64, 1))}),
    ("negative extent", {"q": array("bfloat16", (-3, 4, 64))}),
    ("too large", {"q": array("bfloat16", (2 ** 40, 2 ** 20, 64), (64, 64, 1))}),
    ("tables has 2 rows, q 3", {"tables": array("int32", (2, 5))}),
    ("tables cannot be int64", {"tables": array("int64", (3, 5))}),
    ("over 2\\^31 - 1025 tokens", {"tables": array("int32", (3, 2 ** 28))}),
    ("lengths has 4 entries", {"lengths": array("int32", (4,))}),
    ("lengths is missing", {"lengths": None}),
    ("out cannot be float32", {"out": array("float32", (3, 4, 64))}),
    ("out must have q's shape", {"out": array("bfloat16", (3, 2, 64))}),
    ("must not be a broadcast", {"out": array("bfloat16", (3, 4, 64), (0, 64, 1))}),
    ("lse must be", {"lse": array("float32", (3, 2))}),
    ("lse cannot be bfloat16", {"lse": array("bfloat16", (3, 4))}),
    ("scale must be finite", {"scale": float("nan")}),
    ("scale must be finite", {"scale": -1e39}),
    ("window must not be negative", {"window": -1}),
    ("the cache is missing", {"cache": None}),
    ("one type", {"cache": cache(v=array("float16", (4, 16, 2, 64)))}),
    ("one shape", {"cache": cache(v=array("bfloat16", (4, 16, 2, 32)))}),
    ("k_cache must have 4 dimensions", {"cache": cache(k=array("bfloat16", (64, 2, 64)))}),
    ("k_cache cannot be int32", {"cache": cache(k=array("int32", (4, 16, 2, 64)))}),
    ("has no k_scale", {"cache": cache(k_scale=array("float32", (4, 16, 2)))}),
    ("head_dim 512 is over 256", {"cache": cache(dim=512)}),
    ("must be positive", {"cache": cache(page_size=0)}),
    ("at most 2\\^31 - 1 tokens", {"cache": cache(pages=2 ** 28)}),
])
def test_attention_refuses(match, other):
    attend(match, **other)


def test_scales_are_checked():
    missing = cache("int8")
    missing.v_scale = MtArray()
    attend("needs v_scale", cache=missing)
    attend("k_scale must be", cache=cache("int8", k_scale=array("float32", (4, 16, 3))))
    attend("k_scale cannot be float16", cache=cache("int8", k_scale=array("float16", (4, 16, 2))))


@pytest.mark.parametrize("match,k,v,c,slots", [
    ("k and v are both needed", array("float32", (7, 2, 64)), None, cache(), array("int64", (7,))),
    ("must have one type", array("float32", (7, 2, 64)), array("float16", (7, 2, 64)), cache(), array("int64", (7,))),
    ("as the cache's heads are", array("float32", (7, 3, 64)), array("float32", (7, 3, 64)), cache(), array("int64", (7,))),
    ("k has 7 tokens, slots 8", array("float32", (7, 2, 64)), array("float32", (7, 2, 64)), cache(), array("int64", (8,))),
    ("slots cannot be float32", array("float32", (7, 2, 64)), array("float32", (7, 2, 64)), cache(), array("float32", (7,))),
    ("k cannot be int8", array("int8", (7, 2, 64)), array("int8", (7, 2, 64)), cache(), array("int64", (7,))),
    ("k_cache is written", array("float32", (7, 2, 64)), array("float32", (7, 2, 64)),
     cache(k=array("bfloat16", (4, 16, 2, 64), (0, 128, 64, 1))), array("int64", (7,))),
    ("v_scale is written", array("float32", (7, 2, 64)), array("float32", (7, 2, 64)),
     cache("int8", v_scale=array("float32", (4, 16, 2), (32, 2, 0))), array("int64", (7,))),
    ("over 2\\^31 - 1 rows", array("float32", (2 ** 30, 2, 64)), array("float32", (2 ** 30, 2, 64)), cache(),
     array("int64", (2 ** 30,))),
])
def test_write_refuses(match, k, v, c, slots):
    refused(backend.lib().mt_cache_write(0, k, v, c, slots, None), match)


def test_read_refuses():
    L, slots = backend.lib(), array("int32", (7,))
    rows = array("float32", (7, 2, 64))
    refused(L.mt_cache_read(0, cache(), slots, None, None, None), "k and v are missing")
    refused(L.mt_cache_read(0, cache(), slots, rows, array("float32", (7, 2, 64), (0, 64, 1)), None), "must not be a broadcast")
    refused(L.mt_cache_read(0, cache(), slots, None, array("float32", (8, 2, 64)), None), "v has 8 tokens")
    refused(L.mt_cache_read(0, None, slots, rows, rows, None), "cache is missing")


def test_nothing_to_do_needs_no_device():
    L, need = backend.lib(), ctypes.c_uint64(9)
    none = array("float32", (0, 2, 64), ptr=0)
    assert L.mt_cache_write(0, none, none, cache(), array("int64", (0,), ptr=0), None) == 0
    assert L.mt_cache_read(0, cache(), array("int64", (0,), ptr=0), none, none, None) == 0
    q = array("bfloat16", (0, 4, 64), ptr=0)
    assert L.mt_paged_attention(0, q, cache(), array("int32", (0, 5), ptr=0), array("int32", (0,), ptr=0), q, None,
                                0.125, 0, None, 0, None) == 0
    assert L.mt_paged_attention_workspace(0, q, cache(), array("int32", (0, 5), ptr=0), 0, ctypes.byref(need)) == 0
    assert need.value == 0


def test_device_arrays_only():
    torch = pytest.importorskip("torch")
    import metellus_b200 as mt

    x, i = torch.zeros((2, 2, 64)), torch.zeros(2, dtype=torch.int32)
    c = torch.zeros((4, 16, 2, 64))
    with pytest.raises(ValueError, match="CUDA device"):
        mt.cache_write(x, x, c, c, i)
    with pytest.raises(ValueError, match="CUDA device"):
        mt.paged_attention(x, c, c, i[:, None], i)
    with pytest.raises(TypeError, match="must be a CUDA tensor, not list"):
        mt.cache_read([1], c, i)


def test_arrays_without_the_exchange_api():
    """A tensor whose type has no such interface is told so, not that it is no tensor."""
    pytest.importorskip("torch")
    import metellus_b200 as mt

    class Tensor:
        def __dlpack__(self, **_):
            raise AssertionError("not asked for")

    with pytest.raises(TypeError, match="k_cache is a Tensor, whose type does not offer DLPack's C exchange API"):
        mt.cache_read(Tensor(), Tensor(), Tensor())
