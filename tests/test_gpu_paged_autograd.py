"""The paged cache's operators beside torch's autograd: no derivative is dropped silently, and what they
write counts as modified."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from metellus_b200 import cache_read, cache_write, paged_attention

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(autouse=True)
def _device(cuda_device):
    torch.manual_seed(3)


def arrays():
    a = {"q": torch.randn((2, 4, 64), device=DEV), "k": torch.randn((2, 2, 64), device=DEV),
         "v": torch.randn((2, 2, 64), device=DEV), "out": torch.zeros((2, 4, 64), device=DEV),
         "out_k": torch.zeros((2, 2, 64), device=DEV), "out_v": torch.zeros((2, 2, 64), device=DEV),
         "k_scale": torch.rand((4, 16, 2), device=DEV), "v_scale": torch.rand((4, 16, 2), device=DEV)}
    for name in ("k_cache", "v_cache"):
        a[name] = torch.randint(-100, 100, (4, 16, 2, 64), device=DEV, dtype=torch.int8)
    return a


def int32(*x):
    return torch.tensor(x, device=DEV, dtype=torch.int32)


def attend(a):
    return paged_attention(a["q"], a["k_cache"], a["v_cache"], int32([0, 1], [2, 3]), int32(20, 30), k_scale=a["k_scale"],
                           v_scale=a["v_scale"], out=a["out"])


def write(a):
    return cache_write(a["k"], a["v"], a["k_cache"], a["v_cache"], int32(3, 7), k_scale=a["k_scale"], v_scale=a["v_scale"])


def read(a):
    return cache_read(a["k_cache"], a["v_cache"], int32(3, 7), k_scale=a["k_scale"], v_scale=a["v_scale"],
                      out=(a["out_k"], a["out_v"]))


CALLS = [(attend, ("q", "k_scale", "v_scale", "out")), (write, ("k", "v", "k_scale", "v_scale")),
         (read, ("k_scale", "v_scale", "out_k", "out_v"))]


@pytest.mark.parametrize("call,names", CALLS)
def test_gradients_are_refused(call, names):
    for name in names:
        a = arrays()
        a[name].requires_grad_()
        before = {n: x.detach().clone() for n, x in a.items()}
        with pytest.raises(ValueError, match="requires a gradient"):
            call(a)
        assert all(torch.equal(a[n], before[n]) for n in a)
        with torch.no_grad():
            call(a)


@pytest.mark.parametrize("call,names", CALLS)
def test_tangents_are_refused(call, names):
    for name in names:
        a = arrays()
        with forward_ad.dual_level():
            a[name] = forward_ad.make_dual(a[name], torch.ones_like(a[name]))
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(ValueError, match="has a tangent"):
                    call(a)
            call(arrays())


def test_transforms_are_refused():
    a = arrays()

    def f(q):
        return attend({**a, "q": q, "out": None})

    for run in (lambda: torch.func.jvp(f, (a["q"],), (a["q"],)), lambda: torch.func.grad(lambda q: f(q).sum())(a["q"]),
                lambda: torch.func.vmap(f)(a["q"][None])):
        with pytest.raises((ValueError, RuntimeError)):
            run()


def test_writes_are_counted():
    a = arrays()
    was = {n: x._version for n, x in a.items()}
    attend(a), write(a), read(a)
    written = {"out", "k_cache", "v_cache", "k_scale", "v_scale", "out_k", "out_v"}
    assert {n for n, x in a.items() if x._version > was[n]} == written
    # what was kept for a backward pass, and written over since, is found out there
    x = torch.randn((2, 4, 64), device=DEV, requires_grad=True)
    y = (x * a["out"]).sum()
    attend(a)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        b = arrays()
        attend(b), write(b), read(b)
