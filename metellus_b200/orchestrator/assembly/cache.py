"""Ops on paged key-value caches: one native kernel each (``mt_cache_write``, ``mt_cache_read``,
``mt_paged_attention``), no counterpart in the reference. Slots: the op's tensors in the
order of its C entry point, then the cache's arrays (keys ``<cache>.k`` and so on, which the
runtime binds to the ``PagedCache``'s buffers)."""

from __future__ import annotations

from metellus_b200.compute.fragments import CodegenContext
from metellus_b200.orchestrator.assembly.decision import DecisionView
from metellus_b200.orchestrator.assembly.extras import param_decl
from metellus_b200.orchestrator.ir import CacheReadOp, CacheWriteOp, PagedAttentionOp, rows_of_heads
from metellus_b200.orchestrator.kernel_group import KernelGroup
from metellus_b200.runtime.program import ArraySpec, NativeKernel


def cache_keys(name: str, paged) -> tuple[str, ...]:
    """Env keys of a cache's arrays."""
    return tuple(f"{name}.{part}" for part in paged.parts)


def _heads(what: str, t, heads, head_dim: int) -> ArraySpec:
    rows, n, strides = rows_of_heads(what, t, heads, head_dim)
    return ArraySpec("float32", (rows, n, head_dim), strides)


def assemble_cache_op(decision: DecisionView, function_name: str | None) -> KernelGroup:
    op = decision.ops[0]
    paged = op.paged
    if isinstance(op, CacheWriteOp):
        tensors, entry = (op.k, op.v, op.slots), "mt_cache_write"
        specs = tuple(_heads(entry, t, paged.kv_heads, paged.head_dim) for t in (op.k, op.v))
        specs += (ArraySpec("int32", op.slots.shape, (op.slots.row_stride,)),)
        params = (paged, specs)
    elif isinstance(op, CacheReadOp):
        tensors, entry = (op.slots, op.out), "mt_cache_read"
        heads, rows, dim = op.out.shape
        params = (paged, (ArraySpec("int32", op.slots.shape, (op.slots.row_stride,)),
                          ArraySpec("float32", (rows, heads, dim), (dim, rows * dim, 1))), op.part)
    else:
        assert isinstance(op, PagedAttentionOp)
        tensors, entry = (op.q, op.tables, op.lengths, op.out), "mt_paged_attention"
        params = (paged, (_heads(entry, op.q, None, paged.head_dim),
                          ArraySpec("int32", op.tables.shape, (op.tables.row_stride, op.tables.col_stride)),
                          ArraySpec("int32", op.lengths.shape, (op.lengths.row_stride,)),
                          _heads(entry, op.out, None, paged.head_dim)), op.scale, op.window)
    keys = tuple(t.buffer_key for t in tensors) + cache_keys(op.cache.buffer_key, paged)
    ctx = CodegenContext(function_name=function_name or f"{decision.strategy.value}_{op.out.name}",
                         buffers=tuple(param_decl(k) for k in keys), dims=(), tg_x=1, tg_y=1)
    return KernelGroup(kernel=NativeKernel(entry, params, ctx), bindings=keys, dims=(), grid=(1, 1, 1), threads=(1, 1, 1),
                       ops=decision.ops, strategy=decision.strategy, pipe="native")
