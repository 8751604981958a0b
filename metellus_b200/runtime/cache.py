"""A paged key-value cache in device memory, for programs.

No counterpart in the reference. ``PagedCache`` owns the arrays that
``Operations.cache_write`` / ``cache_read`` / ``paged_attention`` work on. They live as
long as the object does, across calls and across programs that declare it: a prompt's
program and the decode step's share one cache::

    cache = PagedCache(pages=512, page_size=16, kv_heads=8, head_dim=128, dtype="int8")
    ops.cache(cache, "kv")

The device memory is allocated, and zeroed, when a program first runs on it.
"""

from __future__ import annotations

from metellus_b200.runtime import backend
from metellus_b200.runtime.backend import ARRAY_DTYPES, MtArray, MtPagedCache
from metellus_b200.runtime.buffer import Buffer

CACHE_DTYPES = ("float32", "float16", "bfloat16", "int8", "float8_e4m3fn")
_ITEM = {"float32": 4, "float16": 2, "bfloat16": 2, "int8": 1, "float8_e4m3fn": 1}


def device_array(handle: int, dtype: str, shape: tuple[int, ...], strides: tuple[int, ...]) -> MtArray:
    """A buffer as the C entry points take arrays (strides in elements)."""
    return MtArray(backend.buffer_ptr(handle), ARRAY_DTYPES[dtype], len(shape), tuple(shape), tuple(strides))


class PagedCache:
    """``pages`` pages of ``page_size`` tokens of ``kv_heads`` heads, each a row of
    ``head_dim`` keys and one of values. ``int8`` and ``float8_e4m3fn`` caches keep a
    float32 scale per token and head beside each row."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: str = "float32",
                 device: int | None = None) -> None:
        if dtype not in CACHE_DTYPES:
            raise ValueError(f"PagedCache: dtype {dtype!r} is not one of {CACHE_DTYPES}")
        for name, n in (("pages", pages), ("page_size", page_size), ("kv_heads", kv_heads), ("head_dim", head_dim)):
            if not isinstance(n, int) or n < 1:
                raise ValueError(f"PagedCache: {name} must be a positive whole number, got {n!r}")
        if head_dim > 256:
            raise ValueError(f"PagedCache: head_dim {head_dim} is over 256")
        if pages * page_size > 2 ** 31 - 1 or kv_heads > 65535:
            raise ValueError("PagedCache: at most 2^31 - 1 tokens of 65535 heads")
        self.pages, self.page_size, self.kv_heads, self.head_dim = pages, page_size, kv_heads, head_dim
        self.dtype = dtype
        self.device = device
        self._buffers: dict[str, Buffer] = {}

    @property
    def slots(self) -> int:
        return self.pages * self.page_size

    @property
    def parts(self) -> tuple[str, ...]:
        """Names of its arrays, in the order kernels take them."""
        return ("k", "v", "k_scale", "v_scale") if _ITEM[self.dtype] == 1 else ("k", "v")

    def part_bytes(self, part: str) -> int:
        rows = self.slots * self.kv_heads
        return rows * 4 if part.endswith("scale") else rows * self.head_dim * _ITEM[self.dtype]

    def buffer(self, part: str) -> Buffer:
        if part not in self._buffers:
            self._buffers[part] = Buffer.zeros(self.part_bytes(part), self.device)
        return self._buffers[part]

    def descriptor(self, handles: list[int]) -> MtPagedCache:
        """The C description of the arrays whose buffer handles (in ``parts`` order) are given."""
        shape = (self.pages, self.page_size, self.kv_heads)
        outer = (self.page_size * self.kv_heads, self.kv_heads, 1)
        rows = tuple(s * self.head_dim for s in outer) + (1,)
        c = MtPagedCache()
        for part, h in zip(self.parts, handles, strict=True):
            if part.endswith("scale"):
                setattr(c, part, device_array(h, "float32", shape, outer))
            else:
                setattr(c, part, device_array(h, self.dtype, shape + (self.head_dim,), rows))
        return c

    def release(self) -> None:
        """Give the device memory back (a program that runs on the cache afterwards starts from
        zeros)."""
        for b in self._buffers.values():
            b.release()
        self._buffers.clear()

    def __repr__(self) -> str:
        return (f"PagedCache(pages={self.pages}, page_size={self.page_size}, kv_heads={self.kv_heads}, "
                f"head_dim={self.head_dim}, dtype={self.dtype!r})")
