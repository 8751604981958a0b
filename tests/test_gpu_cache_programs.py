"""Programs on paged key-value caches, run by ``run`` and ``Executable``, against numpy in 64
bits over the rows as they were written."""

from __future__ import annotations

import numpy as np
import pytest

from metellus_b200 import Executable, Operations, PagedCache, run
from metellus_b200.runtime import backend

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, PS, WIDTH = 8, 2, 64, 16, 6


@pytest.fixture(autouse=True)
def _device(cuda_device):
    pass


def attend(q, K, V):
    """q (heads, dim); K, V (tokens, kv, dim), float64."""
    g = q.shape[0] // K.shape[1]
    out = np.zeros(q.shape)
    for h in range(q.shape[0]):
        s = K[:, h // g] @ q[h] / np.sqrt(q.shape[1])
        p = np.exp(s - s.max())
        out[h] = p @ V[:, h // g] / p.sum()
    return out


def prompt_program(cache, k, v, slots):
    ops = Operations()
    ops.cache(cache, "kv")
    ops.from_numpy(k, "k")
    ops.from_numpy(v, "v")
    ops.indices(slots, "slots")
    ops.cache_write(k="k", v="v", cache="kv", slots="slots", out="kv1")
    return ops


def step_program(cache, w, batch, model):
    """Projections, the new rows into the cache, attention over it, output projection, residual."""
    ops = Operations()
    ops.cache(cache, "kv")
    ops.from_numpy(np.zeros((batch, model), np.float32), "x")
    for name in ("q", "k", "v"):
        ops.from_numpy(w[name], "w" + name)
        ops.matmul(a="x", b="w" + name, out=name)
    ops.from_numpy(w["o"], "wo")
    ops.indices(np.arange(batch, dtype=np.int32), "slots")
    ops.indices(np.zeros((batch, WIDTH), np.int32), "tables")
    ops.indices(np.zeros(batch, np.int32), "lengths")
    ops.cache_write(k="k", v="v", cache="kv", slots="slots", out="kv1")
    ops.paged_attention(q="q", cache="kv1", tables="tables", lengths="lengths", out="att")
    ops.matmul(a="att", b="wo", out="y")
    ops.elementwise("add", out="out", operands=("y", "x"))
    return ops


# float32: fp32 arithmetic in the chain (matmuls to 1e-6); the others are the cache's rounding: a row's
# error relative to its values at most 2^-8 (bf16), 1 / 254 of its largest (int8), 2^-4 (e4m3)
@pytest.mark.parametrize("dtype,tol", [("float32", 1e-5), ("bfloat16", 1e-2), ("int8", 3e-2), ("float8_e4m3fn", 8e-2)])
def test_prompt_then_steps(dtype, tol):
    """A prompt's program fills the cache, the step's program (replayed from a CUDA graph from its
    second call on) writes and attends with new tables, slots and lengths each time."""
    r = np.random.default_rng(3)
    batch, model = 3, 128
    prompt = [20, 1, 37]
    cache = PagedCache(batch * WIDTH, PS, KV, DIM, dtype)
    tables = r.permutation(batch * WIDTH).astype(np.int32).reshape(batch, WIDTH)
    w = {n: (r.normal(0, 1, (model, m)) / np.sqrt(model)).astype(np.float32)
         for n, m in (("q", HEADS * DIM), ("k", KV * DIM), ("v", KV * DIM))}
    w["o"] = (r.normal(0, 1, (HEADS * DIM, model)) / np.sqrt(HEADS * DIM)).astype(np.float32)

    def slot(b, t):
        return int(tables[b, t // PS]) * PS + t % PS

    K = [r.normal(0, 1, (n, KV, DIM)).astype(np.float32) for n in prompt]
    V = [r.normal(0, 1, (n, KV, DIM)).astype(np.float32) for n in prompt]
    slots = np.array([slot(b, t) for b, n in enumerate(prompt) for t in range(n)] + [-1, -1], np.int32)
    pad = np.zeros((2, KV, DIM), np.float32)
    run(prompt_program(cache, np.concatenate(K + [pad]), np.concatenate(V + [pad]), slots))

    exe = Executable(step_program(cache, w, batch, model), outputs=("out", "att"))
    for i in range(6):
        x = r.normal(0, 1, (batch, model)).astype(np.float32)
        at = [n + i for n in prompt]
        got = exe({"x": x, "slots": np.array([slot(b, t) for b, t in enumerate(at)], np.int32),
                   "tables": tables, "lengths": np.array([t + 1 for t in at], np.int32)})
        q, k, v = ((x.astype(np.float64) @ w[n]).reshape(batch, -1, DIM) for n in ("q", "k", "v"))
        want = np.zeros((batch, HEADS, DIM))
        for b in range(batch):
            K[b], V[b] = np.concatenate([K[b], k[b][None]]), np.concatenate([V[b], v[b][None]])
            want[b] = attend(q[b], K[b].astype(np.float64), V[b].astype(np.float64))
        want = want.reshape(batch, -1)
        assert np.linalg.norm(got["att"] - want) <= tol * np.linalg.norm(want)
        out = want @ w["o"] + x
        assert np.linalg.norm(got["out"] - out) <= tol * np.linalg.norm(out)
    exe.close()

    # the rows back, as batched matrices, through a third program on the same cache
    ops = Operations()
    ops.cache(cache, "kv")
    back = np.array([slot(2, t) for t in range(len(K[2]))] + [-1], np.int32)
    ops.indices(back, "slots")
    ops.cache_read("kv", "slots", out="K")
    ops.cache_read("kv", "slots", out="V", part="v")
    res = run(ops)
    for name, rows in (("K", K[2]), ("V", V[2])):
        got, want = res.env[name], rows.transpose(1, 0, 2)
        assert got.shape == (KV, len(back), DIM) and not got[:, -1].any()
        limit = {"float32": 0, "bfloat16": 2.0 ** -8, "float8_e4m3fn": 2.0 ** -4}.get(dtype)
        # int8: half a step of the row's largest over 127; e4m3: below its normal range half of 2^-9 steps
        largest = np.abs(want).max(-1, keepdims=True)
        bound = largest / 254 * 1.001 if dtype == "int8" else limit * np.abs(want) + (largest / 448 * 2.0 ** -10 if dtype == "float8_e4m3fn" else 0)
        if dtype == "float32":  # the program's own products differ from numpy's by their rounding
            bound = 1e-5 * largest
        assert (np.abs(got[:, :-1] - want) <= bound * 1.01 + 1e-5 * largest).all()
    cache.release()


def test_reading_a_prefix_into_attention():
    """A prompt's second chunk against its first, read back into the batched attention kernel."""
    r = np.random.default_rng(5)
    n, m = 64, 128
    cache = PagedCache(16, PS, KV, DIM, "float32")
    k, v = (r.normal(0, 1, (n, KV, DIM)).astype(np.float32) for _ in range(2))
    q = r.normal(0, 1, (KV, m, DIM)).astype(np.float32)
    slots = r.permutation(16 * PS)[:n].astype(np.int32)
    run(prompt_program(cache, k, v, slots))
    ops = Operations()
    ops.cache(cache, "kv")
    ops.indices(slots, "slots")
    ops.from_numpy(q, "Q")
    ops.cache_read("kv", "slots", out="K")
    ops.cache_read("kv", "slots", out="V", part="v")
    ops.transpose("K", out="Kt")
    ops.matmul(a="Q", b="Kt", out="S")
    ops.elementwise("mul", out="Ss", operands=("S", 0.125))
    ops.reduction("max", out="m", x="Ss")
    ops.reshape("m", (KV, m, 1), out="m2")
    ops.elementwise("subtract", out="Sc", operands=("Ss", "m2"), y_broadcast="col")
    ops.elementwise("exp", out="E", operands=("Sc",))
    ops.reduction("sum", out="l", x="E")
    ops.reshape("l", (KV, m, 1), out="l2")
    ops.elementwise("div", out="P", operands=("E", "l2"), y_broadcast="col")
    ops.matmul(a="P", b="V", out="O")
    res = run(ops)
    s = np.einsum("hmd,nhd->hmn", q.astype(np.float64), k.astype(np.float64)) * 0.125
    p = np.exp(s - s.max(-1, keepdims=True))
    want = np.einsum("hmn,nhd->hmd", p / p.sum(-1, keepdims=True), v.astype(np.float64))
    assert np.linalg.norm(res.env["O"] - want) <= 1e-5 * np.linalg.norm(want)


def test_profile_times_native_ops():
    cache = PagedCache(4, PS, KV, DIM, "int8")
    k = np.ones((5, KV, DIM), np.float32)
    ops = prompt_program(cache, k, k, np.arange(5, dtype=np.int32))
    res = run(ops, profile=True)
    assert res.env["t_0"] > 0


def test_a_released_cache_is_refused():
    cache = PagedCache(4, PS, KV, DIM)
    k = np.ones((5, KV, DIM), np.float32)
    exe = Executable(prompt_program(cache, k, k, np.arange(5, dtype=np.int32)), outputs=())
    exe()
    exe()
    with pytest.raises(ValueError, match="holds a slot twice"):
        exe({"slots": np.array([1, 2, 3, 3, 4], np.int32)})
    with pytest.raises(ValueError, match="must be int32"):
        exe({"slots": np.arange(5)})
    cache.release()
    with pytest.raises(RuntimeError, match="released"):
        exe()
    exe.close()
    backend.sync()


def test_results_repeat():
    """The same call gives the same bits (cuts and joins depend on the lengths alone)."""
    r = np.random.default_rng(7)
    cache = PagedCache(300, PS, KV, DIM, "bfloat16")
    n = 300 * PS
    k = r.normal(0, 1, (n, KV, DIM)).astype(np.float32)
    run(prompt_program(cache, k, k[::-1].copy(), np.arange(n, dtype=np.int32)))
    ops = Operations()
    ops.cache(cache, "kv")
    ops.from_numpy(r.normal(0, 1, (2, HEADS, DIM)).astype(np.float32), "q")
    ops.indices(np.arange(300, dtype=np.int32).reshape(2, 150), "tables")
    ops.indices(np.array([2400, 1777], np.int32), "lengths")
    ops.paged_attention("q", "kv", "tables", "lengths", out="o")
    exe = Executable(ops)
    first = exe()["o"]
    for _ in range(5):
        np.testing.assert_array_equal(exe()["o"], first)
    exe.close()


def test_views_of_index_tensors():
    """Slots that are a view of a matrix: written by, and given back, as int32, by both ways to run."""
    grid = np.array([[7, 2, 40], [33, 5, -1]], np.int32)
    rows = np.random.default_rng(1).normal(0, 1, (6, KV, DIM)).astype(np.float32)

    def program(cache):
        ops = Operations()
        ops.cache(cache, "kv")
        ops.from_numpy(rows, "k")
        ops.indices(grid, "grid")
        ops.reshape("grid", (6,), out="slots")
        ops.transpose("grid", out="turned")
        ops.cache_write(k="k", v="k", cache="kv", slots="slots", out="kv1")
        ops.cache_read("kv1", "slots", out="K")
        return ops

    want = np.where((grid.reshape(-1) >= 0)[:, None, None], rows, 0).transpose(1, 0, 2)
    env = run(program(PagedCache(4, PS, KV, DIM))).env
    assert env["slots"].dtype == np.int32 and np.array_equal(env["slots"], grid.reshape(-1))
    assert env["turned"].dtype == np.int32 and np.array_equal(env["turned"], grid.T)
    assert np.array_equal(env["K"], want)

    exe = Executable(program(PagedCache(4, PS, KV, DIM)), outputs=("K", "grid"))
    for _ in range(3):
        got = exe({"grid": grid})
        assert got["grid"].dtype == np.int32 and np.array_equal(got["grid"], grid)
        assert np.array_equal(got["K"], want)
    with pytest.raises(ValueError, match="must be int32"):
        exe(out={"grid": np.empty((2, 3), np.float32)})
    exe.close()
