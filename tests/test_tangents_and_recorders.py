"""Calls of the operators beside the linears with a forward-mode tangent, and under what writes torch operations down to run them again: their kernels are no torch
operations, so that such a call is a node of its own, or refused, and never an empty output without a word."""
import contextlib

import pytest
import torch
import torch.autograd.forward_ad as fwad
from torch.fx.experimental.proxy_tensor import make_fx

from bitween_b200 import RotaryPositions
from bitween_b200.kernels import _lib


class _Library:
    """Stands for the library: remembers which entry points were called."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append(name) or 0


@pytest.fixture
def library(monkeypatch):
    """The Python path on CPU tensors, launches left out."""
    stub = _Library()
    monkeypatch.setattr(_lib, "_operators", _lib._NoOperators)
    monkeypatch.setattr(_lib, "lib", lambda: stub)
    monkeypatch.setattr(_lib, "require_cuda", lambda t, name: t)
    monkeypatch.setattr(_lib, "on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "raw_stream", lambda device: 0)
    return stub


def _tangent_refused(call, x):
    for mode in (contextlib.nullcontext, torch.no_grad):
        with fwad.dual_level(), mode(), pytest.raises(NotImplementedError, match="jvp"):
            call(fwad.make_dual(x, torch.ones_like(x)))


def _not_recorded(call, x):
    """(a graph of torch operations would hold the output's allocation alone)"""
    for how in ("real", "fake"):
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            make_fx(call, tracing_mode=how)(x)


def _traced(call, x):
    with pytest.warns(torch.jit.TracerWarning):
        return torch.jit.trace(call, x, check_trace=False)


def test_rotate(library):
    r = RotaryPositions(64, 50, device="cpu")
    p, x = torch.arange(3), torch.randn(3, 2, 64).half()
    for call in (lambda x: r.rotate(p, x), lambda x: r.rotate(p, x, x[:, :1])[1]):
        _tangent_refused(call, x)
        _not_recorded(call, x)
        traced = _traced(call, x)
        assert "^RotateFunction" in str(traced.graph) and "aten::empty" not in str(traced.graph)
        library.calls.clear()
        traced(x)
        assert library.calls == ["bw_rotate"]
        # run again with other tensors, which are checked as a call's are
        library.calls.clear()
        for bad in (x.double(), x[:2], x[..., :32]):
            with pytest.raises(Exception, match="must"):
                traced(bad)
        assert not library.calls


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_a_traced_rotate_runs_again_on_other_tensors():
    r = RotaryPositions(64, 50, sections=(8, 12, 12))
    g = torch.Generator(device="cuda").manual_seed(1)
    p = torch.randint(0, 50, (3, 2, 5), generator=g, device="cuda")
    x, other = (torch.randn(2, 5, 4, 64, generator=g, device="cuda").half() for _ in range(2))
    traced = torch.jit.trace(lambda p, x, y: r.rotate(p, x, y), (p, x, other), check_trace=False)
    strided = torch.randn(64, 4, 5, 2, generator=g, device="cuda").half().permute(3, 2, 1, 0)
    for a in (x, other, strided, other.transpose(0, 1).contiguous().transpose(0, 1)):
        for at in (p, p.flip(0)):
            assert all(torch.equal(got, want) for got, want in zip(traced(at, a, x), r.rotate(at, a, x)))
    leaf = other.clone().requires_grad_()
    (got,) = torch.autograd.grad(traced(p, leaf, x)[0], leaf, x)
    (want,) = torch.autograd.grad(r.rotate(p, leaf), leaf, x)
    assert torch.equal(got, want)
    with fwad.dual_level(), pytest.raises(NotImplementedError):
        r.rotate(p, fwad.make_dual(x, x))
    _not_recorded(lambda x: r.rotate(p, x), x)
