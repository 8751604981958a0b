"""A paged key-value cache and the attention that reads it, on device arrays the caller
owns.

The reference's attention reads K and V as whole tensors whose length is fixed when the
program is planned. Generating text needs the step after that: one new token per sequence
against keys and values kept from before. Three operators do it::

    cache_write(k, v, k_cache, v_cache, slots)                # this step's new rows
    out = paged_attention(q, k_cache, v_cache, tables, lengths)
    k, v = cache_read(k_cache, v_cache, slots)                # back, as whole rows

A cache is two arrays ``[pages, page_size, kv_heads, head_dim]`` of float32, float16,
bfloat16, int8 or float8_e4m3fn; the 8-bit types have ``k_scale`` and ``v_scale``,
float32 ``[pages, page_size, kv_heads]``, beside them (value = code * scale). Slot ``s``
is token ``s % page_size`` of page ``s // page_size``; token ``t`` of sequence ``b`` is
in page ``tables[b, t // page_size]``.

Arrays are torch CUDA tensors (anything with ``data_ptr``, ``shape``, ``stride``,
``dtype``, ``device``), all on one device; the last dimension is contiguous, the other
strides are free. Calls run on torch's current stream of that device without waiting for
it, allocate only through torch and can be captured into CUDA graphs. What does not fit
raises ``ValueError`` before anything is launched. What the device alone knows is
handled there: slots and pages outside the cache are skipped, lengths are clamped to the
table's width.

Programs of this package reach the same operators through ``Operations.cache`` and
``PagedCache``.
"""

from __future__ import annotations

import ctypes
import sys

from metellus_b200.runtime import backend
from metellus_b200.runtime.backend import ARRAY_DTYPES, MtArray, MtPagedCache

__all__ = ["cache_read", "cache_write", "paged_attention"]


def _array(x, name: str, device) -> MtArray:
    """``x`` as the C ABI takes it; checks that it lives on ``device``."""
    try:
        dtype = ARRAY_DTYPES.get(str(x.dtype).rpartition(".")[2])
        if dtype is None:
            raise ValueError(f"{name} cannot be {x.dtype}")
        shape, strides = x.shape, x.stride()
        if len(shape) > 4:
            raise ValueError(f"{name} has {len(shape)} dimensions")
        if x.device != device or device.type != "cuda":
            raise ValueError(f"{name} is on {x.device}; every array must be on one CUDA device"
                             + (f" ({device})" if device.type == "cuda" else ""))
        return MtArray(x.data_ptr(), dtype, len(shape), tuple(shape), tuple(strides))
    except AttributeError:
        raise TypeError(f"{name} must be a CUDA tensor, not {type(x).__name__}") from None


def _cache(k_cache, v_cache, k_scale, v_scale, device) -> MtPagedCache:
    c = MtPagedCache(_array(k_cache, "k_cache", device), _array(v_cache, "v_cache", device))
    if k_scale is not None:
        c.k_scale = _array(k_scale, "k_scale", device)
    if v_scale is not None:
        c.v_scale = _array(v_scale, "v_scale", device)
    return c


def _device(x, name: str):
    try:
        return x.device
    except AttributeError:
        raise TypeError(f"{name} must be a CUDA tensor, not {type(x).__name__}") from None


def _stream(device) -> int:
    """torch's current stream of the device; its default stream by the name that does not
    mean the backend's own."""
    return sys.modules["torch"].cuda.current_stream(device).cuda_stream or 1


def _no_grad(**arrays) -> None:
    """The operators have no backward pass: refuse to drop a gradient silently."""
    torch = sys.modules.get("torch")
    if torch is not None and torch.is_grad_enabled():
        for name, x in arrays.items():
            if getattr(x, "requires_grad", False):
                raise ValueError(f"{name} requires a gradient; the paged cache's operators have none "
                                 "(use torch.no_grad() or detach it)")


def cache_write(k, v, k_cache, v_cache, slots, *, k_scale=None, v_scale=None) -> None:
    """Store rows ``k[i]``, ``v[i]`` (``[tokens, kv_heads, head_dim]``; float32, float16 or
    bfloat16) in slot ``slots[i]`` (``[tokens]``, int32 or int64).

    Values are rounded to the cache's type. In the 8-bit types each (token, head) row is
    stored as the codes nearest to ``x / scale`` (ties to even) with ``scale`` the
    row's largest magnitude over 127 (int8) or 448 (float8_e4m3fn), in float32; a row
    that holds an infinity or a NaN gets the scale NaN. A slot outside the cache (such as
    -1 for padding) skips its row. Slots must be distinct: a slot given twice is left
    with a mixture of its rows; the others are not affected."""
    _no_grad(k=k, v=v, k_cache=k_cache, v_cache=v_cache)
    device = _device(k, "k")
    ak, av = _array(k, "k", device), _array(v, "v", device)
    cache, at = _cache(k_cache, v_cache, k_scale, v_scale, device), _array(slots, "slots", device)
    backend._check(backend.lib().mt_cache_write(device.index, ak, av, cache, at, _stream(device)))


def cache_read(k_cache, v_cache, slots, *, k_scale=None, v_scale=None, dtype=None, out=None):
    """The rows in ``slots`` (``[tokens]``, int32 or int64) as ``(k, v)``, each
    ``[tokens, kv_heads, head_dim]``; slots outside the cache read as zeros.

    ``dtype`` (default: the cache's type, float32 for the 8-bit ones) is the rows' type;
    ``out=(k, v)`` writes into given tensors instead, of any strides (such as a
    ``[kv_heads, tokens, head_dim]`` tensor's transpose)."""
    _no_grad(k_cache=k_cache, v_cache=v_cache)
    device = _device(k_cache, "k_cache")
    cache, at = _cache(k_cache, v_cache, k_scale, v_scale, device), _array(slots, "slots", device)
    if out is None:
        if cache.k.ndim != 4 or at.ndim != 1:
            raise ValueError("cache_read: k_cache must have 4 dimensions and slots 1")
        shape = (slots.shape[0], k_cache.shape[2], k_cache.shape[3])
        if dtype is None:
            dtype = sys.modules["torch"].float32 if k_scale is not None else k_cache.dtype
        out = (k_cache.new_empty(shape, dtype=dtype), k_cache.new_empty(shape, dtype=dtype))
    elif dtype is not None:
        raise ValueError("cache_read: dtype and out exclude one another")
    k, v = out
    ak, av = _array(k, "out[0]", device), _array(v, "out[1]", device)
    backend._check(backend.lib().mt_cache_read(device.index, cache, at, ak, av, _stream(device)))
    return k, v


def paged_attention(q, k_cache, v_cache, tables, lengths, *, k_scale=None, v_scale=None, scale=None, window=0,
                    out=None, return_lse=False):
    """Attention of one query token per sequence over the cache: for each sequence ``b``
    and head ``h``, ``softmax(scale * q[b, h] . K) @ V`` over its visible tokens.

    ``q``: ``[batch, heads, head_dim]`` of float32, of the cache's own 16-bit type, or of
    any of the three on an 8-bit cache (a float32 cache takes float32). Heads
    ``h * kv_heads // heads`` share a key-value head. ``tables``: int32 ``[batch, width]``; ``lengths``:
    int32 ``[batch]``, the tokens in the cache, this step's own among them. ``scale``
    defaults to ``head_dim ** -0.5``; with ``window`` > 0 only the last ``window`` tokens
    are visible. Returns ``out`` (``q``'s shape and type), and with ``return_lse`` also
    the float32 ``[batch, heads]`` natural logarithms of the sums of ``exp(scores)``, by
    which results over parts of a sequence can be joined. A sequence without visible
    tokens gets zeros (and -inf). Scores, sums and accumulators are float32."""
    _no_grad(q=q, k_cache=k_cache, v_cache=v_cache)
    device = _device(q, "q")
    aq = _array(q, "q", device)
    cache = _cache(k_cache, v_cache, k_scale, v_scale, device)
    at, an = _array(tables, "tables", device), _array(lengths, "lengths", device)
    if out is None:
        out = q.new_empty(q.shape)
    ao = _array(out, "out", device)
    if scale is None:
        scale = float(q.shape[-1]) ** -0.5
    lse = al = None
    if return_lse:
        if aq.ndim != 3:
            raise ValueError(f"paged_attention: q must have 3 dimensions, not {aq.ndim}")
        lse = q.new_empty(q.shape[:2], dtype=sys.modules["torch"].float32)
        al = _array(lse, "lse", device)
    L = backend.lib()
    need = ctypes.c_uint64(0)
    backend._check(L.mt_paged_attention_workspace(device.index, aq, cache, at, window, ctypes.byref(need)))
    space = q.new_empty(need.value, dtype=sys.modules["torch"].uint8) if need.value else None
    backend._check(L.mt_paged_attention(device.index, aq, cache, at, an, ao, al, scale, window,
                                        None if space is None else space.data_ptr(), need.value, _stream(device)))
    return (out, lse) if return_lse else out
