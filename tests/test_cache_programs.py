"""Paged key-value caches in programs: what the builder accepts and refuses, and the plans
(no device)."""

from __future__ import annotations

import numpy as np
import pytest

from metellus_b200 import Operations, PagedCache, compile_program
from metellus_b200.orchestrator.kernel_group import FusionStrategy as S
from metellus_b200.orchestrator.scheduler import schedule
from metellus_b200.runtime.program import BindCache, Dispatch, Free, Unbind


def f32(*shape):
    return np.zeros(shape, np.float32)


def i32(*shape):
    return np.arange(int(np.prod(shape)), dtype=np.int32).reshape(shape)


def step(cache=None):
    """One decode step of one layer: projections, the new rows into the cache, attention over it, the
    output projection with the residual."""
    cache = cache or PagedCache(pages=8, page_size=16, kv_heads=2, head_dim=64, dtype="int8")
    ops = Operations()
    ops.cache(cache, "kv")
    ops.from_numpy(f32(3, 256), "x")
    for name, n in (("wq", 256), ("wk", 128), ("wv", 128)):
        ops.from_numpy(f32(256, n), name)
        ops.matmul(a="x", b=name, out=name[1])
    ops.from_numpy(f32(256, 256), "wo")
    ops.indices(i32(3), "slots")
    ops.indices(i32(3, 4), "tables")
    ops.indices(i32(3), "lengths")
    ops.cache_write(k="k", v="v", cache="kv", slots="slots", out="kv1")
    ops.paged_attention(q="q", cache="kv1", tables="tables", lengths="lengths", out="o")
    ops.matmul(a="o", b="wo", out="y")
    ops.elementwise("add", out="out", operands=("y", "x"))
    return ops


def test_decode_step_plan():
    ops = step()
    groups = compile_program(ops)
    kinds = [g.strategy for g in groups]
    assert kinds.index(S.CACHE_WRITE) < kinds.index(S.PAGED_ATTENTION)
    assert kinds.count(S.CACHE_WRITE) == kinds.count(S.PAGED_ATTENTION) == 1 and len(groups) == 6
    attend = groups[kinds.index(S.PAGED_ATTENTION)]
    assert attend.bindings == ("q", "tables", "lengths", "o", "kv.k", "kv.v", "kv.k_scale", "kv.v_scale")
    # the cache is bound and unbound, never allocated, downloaded or freed
    steps = schedule(ops, groups).fragments
    assert [s.name for s in steps if isinstance(s, BindCache)] == ["kv"]
    assert sorted(s.name for s in steps if isinstance(s, Unbind)) == ["kv.k", "kv.k_scale", "kv.v", "kv.v_scale"]
    assert not any(s.name.startswith("kv") for s in steps if isinstance(s, Free))
    assert [d.kernel.entry for d in steps if isinstance(d, Dispatch) and hasattr(d.kernel, "entry")] == [
        "mt_cache_write", "mt_paged_attention"]


def test_read_feeds_batched_matmul():
    ops = Operations()
    ops.cache(PagedCache(4, 16, 2, 64), "kv")
    ops.indices(i32(20), "slots")
    assert ops.cache_read("kv", "slots", out="K").shape == (2, 20, 64)
    ops.cache_read("kv", "slots", out="V", part="v")
    ops.from_numpy(f32(2, 5, 64), "Q")
    ops.transpose("K", out="Kt")
    ops.matmul(a="Q", b="Kt", out="S")
    assert ops.matmul(a="S", b="V", out="O").shape == (2, 5, 64)
    kinds = [g.strategy for g in compile_program(ops)]
    assert kinds.count(S.CACHE_READ) == 2


def test_row_forms():
    """Rows of heads as (rows, heads * head_dim) and (rows, heads, head_dim)."""
    for shape_k, shape_q in (((3, 128), (3, 512)), ((3, 2, 64), (3, 8, 64))):
        ops = Operations()
        ops.cache(PagedCache(4, 16, 2, 64), "kv")
        ops.from_numpy(f32(*shape_k), "k")
        ops.from_numpy(f32(*shape_q), "q")
        ops.indices(i32(3), "slots")
        ops.indices(i32(3, 2), "tables")
        ops.cache_write(k="k", v="k", cache="kv", slots="slots", out="kv1")
        assert ops.paged_attention(q="q", cache="kv1", tables="tables", lengths="slots", out="o").shape == shape_q


@pytest.mark.parametrize("match,call", [
    ("is not a cache", lambda o: o.cache_write(k="k", v="k", cache="k", slots="slots", out="z")),
    ("not rows of 2 heads of 64", lambda o: o.cache_write(k="q", v="k", cache="kv", slots="slots", out="z")),
    ("must be an int32 tensor of 1", lambda o: o.cache_write(k="k", v="k", cache="kv", slots="tables", out="z")),
    ("must be an int32 tensor of 1", lambda o: o.cache_write(k="k", v="k", cache="kv", slots="k", out="z")),
    ("has 3 rows, 'more' 4", lambda o: o.cache_write(k="k", v="k", cache="kv", slots="more", out="z")),
    ("already exists", lambda o: o.cache_write(k="k", v="k", cache="kv", slots="slots", out="k")),
    ("not declared", lambda o: o.cache_write(k="k", v="k", cache="nope", slots="slots", out="z")),
    ("part must be", lambda o: o.cache_read("kv", "slots", out="z", part="both")),
    ("must be an int32 tensor of 2", lambda o: o.paged_attention("q", "kv", "slots", "slots", out="z")),
    ("q has 3 rows", lambda o: o.paged_attention("q", "kv", "tables", "more", out="z")),
    ("not a multiple of 2", lambda o: o.paged_attention("odd", "kv", "tables", "slots", out="z")),
    ("scale must be finite", lambda o: o.paged_attention("q", "kv", "tables", "slots", out="z", scale=float("inf"))),
    ("window must not", lambda o: o.paged_attention("q", "kv", "tables", "slots", out="z", window=-1)),
    ("is a cache", lambda o: o.transpose("kv", out="z")),
    ("is a cache", lambda o: o.reshape("kv", (4, 2048), out="z")),
    ("float32 tensors", lambda o: o.elementwise("add", out="z", operands=("tables", 1.0))),
    ("float32 tensors", lambda o: o.reduction("sum", out="z", x="tables")),
    ("dtypes must match", lambda o: o.matmul(a="tables", b="tables2", out="z")),
    ("must be int32", lambda o: o.indices(np.zeros(3, np.int64), "z")),
    ("indices\\(\\) takes int32", lambda o: o.from_numpy(f32(3), "slots")),
    ("already declared under another name", lambda o: o.cache(o.caches["kv"], "other")),
    ("already declared", lambda o: o.cache(PagedCache(1, 1, 1, 1), "k")),
    ("contiguous", lambda o: o.cache_write(k="turned", v="k", cache="kv", slots="slots", out="z")),
])
def test_builder_refuses(match, call):
    o = Operations()
    o.cache(PagedCache(4, 16, 2, 64), "kv")
    o.from_numpy(f32(3, 128), "k")
    o.from_numpy(f32(3, 512), "q")
    o.from_numpy(f32(3, 192), "odd")
    o.from_numpy(f32(128, 3), "columns")
    o.transpose("columns", out="turned")
    o.indices(i32(3), "slots")
    o.indices(i32(4), "more")
    o.indices(i32(3, 2), "tables")
    o.indices(i32(2, 3), "tables2")
    before = len(o.build()), set(o.tensors)
    with pytest.raises(ValueError, match=match):
        call(o)
    assert (len(o.build()), set(o.tensors)) == before


def test_only_the_newest_name_of_a_cache():
    o = step()
    with pytest.raises(ValueError, match="newest name is 'kv1'"):
        o.paged_attention("q", "kv", "tables", "lengths", out="z")
    with pytest.raises(ValueError, match="write it first"):
        o.cache_write(k="k", v="v", cache="kv1", slots="slots", out="kv2")


def test_repeated_slots_from_the_host():
    o = Operations()
    o.cache(PagedCache(4, 16, 2, 64), "kv")
    o.from_numpy(f32(4, 128), "k")
    o.indices(np.array([5, -1, 5, -1], np.int32), "slots")
    o.cache_write(k="k", v="k", cache="kv", slots="slots", out="kv1")
    with pytest.raises(ValueError, match="holds a slot twice"):
        schedule(o, compile_program(o))


@pytest.mark.parametrize("kwargs", [dict(dtype="float64"), dict(pages=0), dict(head_dim=257), dict(page_size=-1),
                                    dict(kv_heads=1.5), dict(pages=2 ** 28)])
def test_cache_arguments(kwargs):
    a = dict(pages=4, page_size=16, kv_heads=2, head_dim=64)
    a.update(kwargs)
    with pytest.raises(ValueError):
        PagedCache(**a)


def test_names_of_a_caches_arrays_are_taken():
    ops = Operations()
    ops.cache(PagedCache(4, 16, 2, 64), "kv")
    ops.from_numpy(f32(3, 128), "kv.k")
    ops.indices(i32(3), "slots")
    ops.cache_write(k="kv.k", v="kv.k", cache="kv", slots="slots", out="kv1")
    with pytest.raises(ValueError, match="'kv.k' has the name of an array of cache 'kv'"):
        schedule(ops, compile_program(ops))


def test_views_of_index_tensors_stay_int32():
    """What a plan downloads of an int32 tensor (its views, as of any other) is int32 on the host."""
    from metellus_b200.runtime.program import Download

    ops = Operations()
    ops.cache(PagedCache(4, 16, 2, 64), "kv")
    ops.from_numpy(f32(6, 128), "k")
    ops.indices(i32(2, 3), "grid")
    ops.reshape("grid", (6,), out="slots")
    ops.transpose("grid", out="turned")
    ops.reshape("k", (6, 2, 64), out="rows")
    ops.cache_write(k="k", v="rows", cache="kv", slots="slots", out="kv1")
    steps = schedule(ops, compile_program(ops)).fragments
    got = {s.into: np.dtype(s.dtype) for s in steps if isinstance(s, Download)}
    assert got == {"slots": np.int32, "turned": np.int32, "rows": np.float32}
