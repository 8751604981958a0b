"""A program compiled once and bound to device memory for repeated execution.

``run(ops)`` (reference: src/api/run.py) plans, compiles, allocates, runs and frees on
every call, like the reference. Serving loops and benchmarks call the same program
many times on new inputs; ``Executable`` does the planning and compilation once,
keeps every bound device buffer for its lifetime (a persistent pool for the
program), and replays the dispatch list from a CUDA graph (captured on the second
call, after the first call has loaded every module), so a call costs the input
copies, one graph launch and the output copies. Downloads run on the device's copy
stream, after the kernels and overlapping the next call's uploads (PCIe is full
duplex); the next call's kernels wait for them before overwriting the outputs::

    exe = Executable(ops, outputs=("out",))
    res = exe({"x": x, "y": y, "z": z})          # dict name -> host ndarray
    exe(inputs, out={"out": pinned}, wait=False)  # asynchronous with pinned buffers

Inputs are the program's ``from_numpy`` / ``input`` tensors by name; host arrays in
page-locked memory (``backend.PinnedArray``) copy asynchronously.
"""

from __future__ import annotations

from typing import Iterable

import numpy as np

from metellus_b200.api.run import compile_program
from metellus_b200.orchestrator.builder import Operations
from metellus_b200.orchestrator.kernel_group import STATUS_KEY
from metellus_b200.orchestrator.assembly.cache import cache_keys
from metellus_b200.orchestrator.scheduler import buffer_sizes, check_slots, dispatch_of, host_dtype, scratch_of
from metellus_b200.runtime import backend
from metellus_b200.runtime.buffer import Buffer
from metellus_b200.runtime.program import BindCache, CheckStatus


class Executable:
    def __init__(self, ops: Operations, outputs: Iterable[str] | None = None, *, graph: bool = True,
                 b200: bool = True) -> None:
        self.ops = ops
        self.groups = compile_program(ops, b200=b200)
        tensors = ops.tensors
        program = ops.build()
        produced = {op.out.name for op in program}
        used = {t.name for op in program for t in op.inputs}
        self.outputs = (tuple(outputs) if outputs is not None
                        else tuple(sorted(n for n in produced - used if tensors[n].dtype != "cache")))
        bound = {k for g in self.groups for k in g.bindings}
        for name in self.outputs:
            if name not in tensors:
                raise KeyError(f"Executable: unknown output {name!r}")
            if tensors[name].buffer_key not in bound:
                raise ValueError(f"Executable: {name!r} is fused away (not materialised by the plan)")
        self.input_keys = {name: tensors[name].buffer_key for name in ops.uploads}
        sizes = buffer_sizes(ops, self.groups)
        self.env: dict[str, Buffer] = {}
        self._cache_keys: set[str] = set()
        for name, arr in ops.uploads.items():
            if tensors[name].dtype == "int32":
                check_slots(ops, name, arr)
            self.env[tensors[name].buffer_key] = Buffer.from_numpy(arr)
        # a cache's buffers are its own: bound here, not released with the program
        for name, cache in ops.caches.items():
            BindCache(name=name, cache=cache).execute(self.env)
            self._cache_keys.update(cache_keys(name, cache))
        for k, n in scratch_of(self.groups).items():
            self.env[k] = Buffer.zeros(n)
        for g in self.groups:
            for k in g.bindings:
                if k not in self.env:
                    self.env[k] = Buffer(sizes[k])
        self.dispatches = tuple(dispatch_of(g) for g in self.groups)
        for g in self.groups:
            _ = g.kernel.handle  # compile + load before the first call
        # collectives and the host-timed paths stay out of graphs
        self._graph_ok = graph and not any("nccl" in (g.pipe or "") for g in self.groups)
        self._graph: int | None = None
        self._calls = 0
        self._kernels_done = backend.Event()
        self._read_done = backend.Event()
        self._read_pending = False

    # -- execution ------------------------------------------------------------------

    def _launch(self) -> None:
        for k in self._cache_keys:
            _ = self.env[k].handle  # raises where its cache has been released: the graph holds the address
        if self._graph is not None:
            backend.graph_launch(self._graph)
            return
        if self._graph_ok and self._calls >= 1:
            backend.graph_begin()
            try:
                for d in self.dispatches:
                    d.execute(self.env)
            except Exception:
                try:
                    backend.graph_end()
                except Exception:
                    pass
                self._graph_ok = False
                raise
            self._graph = backend.graph_end()
            backend.graph_launch(self._graph)
            return
        for d in self.dispatches:
            d.execute(self.env)

    def __call__(self, inputs: dict[str, np.ndarray] | None = None, out: dict[str, np.ndarray] | None = None, *,
                 wait: bool = True) -> dict[str, np.ndarray]:
        tensors = self.ops.tensors
        for name, dst in (out or {}).items():
            if name in tensors and tensors[name].dtype == "int32" and dst.dtype != np.int32:
                raise ValueError(f"Executable: destination for {name!r} must be int32, got {dst.dtype}")
        for name, arr in (inputs or {}).items():
            if name not in self.input_keys:
                raise KeyError(f"Executable: {name!r} is not an input of the program")
            if tuple(np.shape(arr)) != tuple(tensors[name].shape):
                raise ValueError(f"Executable: input {name!r} has shape {np.shape(arr)}, "
                                 f"expected {tensors[name].shape}")
            if tensors[name].dtype == "int32":
                arr = np.asarray(arr)
                if arr.dtype != np.int32:
                    raise ValueError(f"Executable: input {name!r} must be int32, got {arr.dtype}")
                check_slots(self.ops, name, arr)
            else:
                arr = np.asarray(arr, dtype=np.float32)
            self.env[self.input_keys[name]].write(arr, wait=False)
        if self._read_pending:  # the previous call's downloads must finish before the outputs change
            backend.stream_wait_event(self._read_done)
        self._launch()
        self._calls += 1
        self._kernels_done.record()
        results: dict[str, np.ndarray] = {}
        for k, name in enumerate(self.outputs):
            t = tensors[name]
            dst = (out or {}).get(name)
            if dst is None:
                dst = np.empty(t.shape, dtype=host_dtype(t))
            if t.buffer_key != t.name:
                raise ValueError(f"Executable: output {name!r} is a view; request its owner {t.buffer_key!r}")
            if dst.nbytes > self.env[t.buffer_key].nbytes or not dst.flags["C_CONTIGUOUS"]:
                raise ValueError(f"Executable: destination for {name!r} is not a contiguous array of its size")
            last = k == len(self.outputs) - 1
            backend.read_buffer_after(self.env[t.buffer_key].handle, dst, after=self._kernels_done,
                                      done=self._read_done if last else None)
            results[name] = dst
        self._read_pending = bool(self.outputs)
        if wait:
            self.synchronize()
        return results

    def join(self) -> None:
        """Order the device's main stream after the pending downloads (no host wait):
        an event recorded on the main stream afterwards covers them."""
        if self._read_pending:
            backend.stream_wait_event(self._read_done)

    def synchronize(self) -> None:
        """Wait for the device (kernels and downloads), then raise if a kernel's bounded
        wait timed out."""
        backend.sync()
        self._read_pending = False
        if STATUS_KEY in self.env:
            CheckStatus(STATUS_KEY).execute(self.env)

    def close(self) -> None:
        if self._graph is not None:
            backend.graph_destroy(self._graph)
            self._graph = None
        for key, b in self.env.items():
            if key not in self._cache_keys:
                b.release()
        self.env.clear()

    def __del__(self) -> None:
        try:
            self.close()
        except Exception:
            pass
