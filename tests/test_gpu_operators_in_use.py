"""Calls of the cache and the adapters as programs around them make them: under autograd, cast modules, and captures beside living graphs."""
import os
import subprocess
import sys

import pytest
import torch

from bitween_b200 import AdaptedLinear, QuantizedKVCache, QuantizedLinear, adapter_matmul
from bitween_b200.kernels import _lib

DEV = "cuda"


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_lib, "_operators", _lib._NoOperators)


def _bank(M=5, K=64, N=32, n=2, r=8):
    g = torch.Generator(device=DEV).manual_seed(3)
    x, down, up = (torch.randn(s, generator=g, device=DEV).half() for s in ((M, K), (n, r, K), (n, r, N)))
    return x, down, up, torch.zeros(M, dtype=torch.int32, device=DEV)


@pytest.mark.gpu
def test_attend_refuses_a_query_that_wants_a_gradient(path):
    cache = QuantizedKVCache(2, 16, 2, 64, bits=4, device=DEV)
    x = torch.randn(3, 2, 64, device=DEV).half().requires_grad_()
    cache.append(x, x, torch.arange(3, device=DEV))
    table, lengths = torch.zeros(3, 1, dtype=torch.int32, device=DEV), torch.full((3,), 3, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="no gradient"):
        cache.attend(x, table, lengths)
    with torch.no_grad():
        quiet = cache.attend(x, table, lengths)
    assert not quiet.requires_grad and torch.equal(quiet, cache.attend(x.detach(), table, lengths))
    assert torch.equal(cache.attend(x.detach(), table, lengths, softmax_scale=torch.tensor(0.125)), quiet)


@pytest.mark.gpu
def test_a_base_written_in_place_is_noticed_by_those_who_saved_it(path):
    x, down, up, index = _bank()
    base = torch.randn(5, 32, device=DEV).half()
    w = torch.randn(5, 32, device=DEV).half().requires_grad_()
    loss = (w * base).sum()
    adapter_matmul(x, down, up, index, base=base, out=base)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        held = torch.randn(5, 32, device=DEV).half()
    before = held.clone()
    adapter_matmul(x, down, up, index, base=held, out=held)
    assert torch.equal(held, adapter_matmul(x, down, up, index, base=before))


@pytest.mark.gpu
def test_an_output_over_the_scaling_or_the_index(path):
    x, down, up, index = _bank(M=64)
    storage = torch.zeros(64 * 32, dtype=torch.float16, device=DEV)
    scaling = storage.view(torch.float32)[:2].fill_(0.5)
    over = storage.view(torch.int32)[512:512 + 64].copy_(index)
    want = adapter_matmul(x, down, up, index, scaling=scaling.clone())
    assert torch.equal(adapter_matmul(x, down, up, over, scaling=scaling, out=storage.view(64, 32)), want)


@pytest.mark.gpu
def test_a_cast_module_keeps_running():
    lin = torch.nn.Linear(64, 32).to(DEV)
    adapted = AdaptedLinear(QuantizedLinear.from_float(lin, bits=4, group_size=32), 2, 8, scaling=0.5)
    with torch.no_grad():
        adapted.up.normal_()
        x, index = torch.randn(5, 64, device=DEV).half(), torch.tensor([0, 1, -1, 0, 1], dtype=torch.int32, device=DEV)
        want = adapted(x, index)
        assert torch.equal(adapted.half()(x, index), want)          # (a scaling of 0.5 is an fp16 number)


def test_widths_beyond_a_grid_are_refused():
    L, P = _lib.lib(), 1 << 20
    assert L.bw_adapter_forward(P, 1, 4, 65535 * 256 + 1, 64, P, P, 2, 5, P, None, None, P, P, 1 << 40, None) == 3
    assert L.bw_adapter_forward(P, 1, 4, 64, 65535 * 256 + 1, P, P, 2, 5, P, None, None, P, P, 1 << 40, None) == 3


@pytest.mark.gpu
def test_a_captured_backward_beside_a_living_graph_of_the_same_leaves():
    """Refused while the graph recorded on the default stream lives; captured once it is gone."""
    program = """
import torch
from bitween_b200 import adapter_matmul
g = torch.Generator(device="cuda").manual_seed(5)
x, down, up = (torch.randn(s, generator=g, device="cuda").half().requires_grad_() for s in ((130, 64), (2, 8, 64), (2, 8, 32)))
index = torch.randint(-1, 2, (130,), generator=g, device="cuda").int()
grad = torch.randn(130, 32, generator=g, device="cuda").half()
want = torch.autograd.grad(adapter_matmul(x, down, up, index), (x, down, up), grad)
living = adapter_matmul(x, down, up, index)
torch.cuda.synchronize()
refused = False
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = adapter_matmul(x, down, up, index)
    try:
        torch.autograd.grad(y, (x, down, up), grad)
    except RuntimeError as e:
        refused = "cannot be captured" in str(e)
assert refused
again = torch.autograd.grad(living, (x, down, up), grad)
assert all(torch.equal(a, b) for a, b in zip(again, want))
del living, y
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = torch.autograd.grad(adapter_matmul(x, down, up, index), (x, down, up), grad)
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("done")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", program], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]
