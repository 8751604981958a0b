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

Arrays are torch CUDA tensors (or another framework's) whose type offers DLPack's C exchange
API, as torch 2.11's does, all on one device; the last dimension is contiguous, the other
strides are free. Calls run on torch's current stream of that device without waiting for
it, allocate only through torch and can be captured into CUDA graphs. What does not fit
raises ``ValueError`` before anything is launched, tensors that require a gradient (or have a
tangent) among it: the operators have no derivatives. Arrays that are written count as modified in
place. What the device alone knows is
handled there: slots and pages outside the cache are skipped, lengths are clamped to the
table's width.

Programs of this package reach the same operators through ``Operations.cache`` and
``PagedCache``.
"""

from __future__ import annotations

import importlib.machinery
import importlib.util
import sys

from metellus_b200.runtime import backend

__all__ = ["cache_read", "cache_write", "paged_attention"]

_module = None


def _native():
    """The binding beside the backend library (built with it by ``metellus_b200.csrc.build``)."""
    global _module
    if _module is None:
        backend.lib()  # reports a missing library, and is the one the binding finds
        path = backend.LIB_PATH.parent / "_metellus_paged.so"
        if not path.exists():
            raise RuntimeError(f"Metellus CUDA backend not built: {path} is missing "
                               "(run `python -m metellus_b200.csrc.build` or __graft_entry__.build())")
        loader = importlib.machinery.ExtensionFileLoader("_metellus_paged", str(path))
        spec = importlib.util.spec_from_loader("_metellus_paged", loader)
        _module = importlib.util.module_from_spec(spec)
        loader.exec_module(_module)
    return _module


_torch = None   # (forward_ad, what the binding is given, the same within forward-mode differentiation)


def _autograd():
    """torch's tensors, and its functions by which the binding refuses tensors with a gradient or a
    tangent and counts writes; None without torch."""
    global _torch
    if _torch is None:
        torch = sys.modules.get("torch")
        if torch is None:
            return None
        forward_ad = torch.autograd.forward_ad
        hooks = (torch.Tensor, torch.is_grad_enabled, torch.autograd.graph.increment_version)
        _torch = (forward_ad, hooks + (None,), hooks + (forward_ad.unpack_dual,))
    forward_ad, plain, dual = _torch
    return dual if getattr(forward_ad, "_current_level", 0) >= 0 else plain


def _dtype_code(dtype) -> int:
    code = backend.ARRAY_DTYPES.get(str(dtype).rpartition(".")[2], -1)
    if not 0 <= code <= 2:
        raise ValueError(f"cache_read: rows are float32, float16 or bfloat16, not {dtype}")
    return code


def cache_write(k, v, k_cache, v_cache, slots, *, k_scale=None, v_scale=None) -> None:
    """Store rows ``k[i]``, ``v[i]`` (``[tokens, kv_heads, head_dim]``; float32, float16 or
    bfloat16) in slot ``slots[i]`` (``[tokens]``, int32 or int64).

    Values are rounded to the cache's type. In the 8-bit types each (token, head) row is
    stored as the codes nearest to ``x / scale`` (ties to even) with ``scale`` the
    row's largest magnitude over 127 (int8) or 448 (float8_e4m3fn), in float32; a row
    that holds an infinity or a NaN gets the scale NaN. A slot outside the cache (such as
    -1 for padding) skips its row. Slots must be distinct: a slot given twice is left
    with a mixture of its rows; the others are not affected."""
    (_module or _native()).cache_write(_autograd(), k, v, k_cache, v_cache, k_scale, v_scale, slots)


def cache_read(k_cache, v_cache, slots, *, k_scale=None, v_scale=None, dtype=None, out=None):
    """The rows in ``slots`` (``[tokens]``, int32 or int64) as ``(k, v)``, each
    ``[tokens, kv_heads, head_dim]``; slots outside the cache read as zeros.

    ``dtype`` (default: the cache's type, float32 for the 8-bit ones) is the rows' type;
    ``out=(k, v)`` writes into given tensors instead, of any strides (such as a
    ``[kv_heads, tokens, head_dim]`` tensor's transpose)."""
    if out is not None and dtype is not None:
        raise ValueError("cache_read: dtype and out exclude one another")
    to_k, to_v = (None, None) if out is None else out
    return (_module or _native()).cache_read(_autograd(), k_cache, v_cache, k_scale, v_scale, slots,
                                             -1 if dtype is None else _dtype_code(dtype), to_k, to_v)


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
    return (_module or _native()).paged_attention(_autograd(), q, k_cache, v_cache, k_scale, v_scale, tables, lengths,
                                                  scale, window, out, return_lse)
