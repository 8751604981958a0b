"""The paged cache's C entry points called by several threads at once, from the first call on."""

from __future__ import annotations

import ctypes
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def calls_from_threads() -> None:
    import threading

    import torch

    from metellus_b200.runtime import backend
    from metellus_b200.runtime.backend import ARRAY_DTYPES, MtArray, MtPagedCache

    def array(x):
        return MtArray(x.data_ptr(), ARRAY_DTYPES[str(x.dtype).rpartition(".")[2]], x.dim(), tuple(x.shape), x.stride())

    torch.manual_seed(2)
    L, threads, batch, width = backend.lib(), 8, 6, 40
    k, v = (torch.randn((batch * width, 16, 2, 64), device="cuda").bfloat16() for _ in range(2))
    q = torch.randn((batch, 8, 64), device="cuda").bfloat16()
    tables = torch.randperm(batch * width, device="cuda").int().view(batch, width)
    lengths = torch.randint(1, width * 16 + 1, (batch,), device="cuda").int()
    outs = [torch.empty_like(q) for _ in range(threads)]
    spaces = [torch.empty(1 << 25, device="cuda", dtype=torch.uint8) for _ in range(threads)]
    streams = [torch.cuda.Stream() for _ in range(threads)]
    torch.cuda.synchronize()
    gate = threading.Barrier(threads)

    def one(i):
        need = ctypes.c_uint64()
        cache = MtPagedCache(array(k), array(v))
        gate.wait()
        for _ in range(20):
            assert L.mt_paged_attention_workspace(0, array(q), cache, array(tables), 0, ctypes.byref(need)) == 0
            assert need.value <= spaces[i].numel()
            assert L.mt_paged_attention(0, array(q), cache, array(tables), array(lengths), array(outs[i]), None, 0.125, 0,
                                        spaces[i].data_ptr(), need.value, streams[i].cuda_stream) == 0

    with ThreadPoolExecutor(threads) as pool:
        list(pool.map(one, range(threads)))
    torch.cuda.synchronize()
    for out in outs:
        assert torch.equal(out, outs[0]) and bool(out.isfinite().all()) and bool(out.any())


def test_threads(cuda_device):
    """In a process of its own: the entry points' set-up is done once, by the threads' first calls."""
    done = subprocess.run([sys.executable, "-c", "from tests.test_gpu_paged_threads import calls_from_threads; calls_from_threads()"],
                          cwd=Path(__file__).parent.parent, timeout=300)
    assert done.returncode == 0
