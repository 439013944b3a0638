"""The native host side of the cache's and the adapters' calls: which calls it takes, that the others go the Python way, and that both are alike."""
import math

import pytest
import torch

from bitween_b200 import QuantizedKVCache, adapter_matmul
from bitween_b200.adapters import AdapterFunction
from bitween_b200.kernels import _lib

DEV = "cuda"


def test_calls_that_are_not_plain_are_left_to_the_python_path():
    ops = _lib.host_operators()
    codes, params = torch.zeros(2, 1, 16, 8, dtype=torch.int32), torch.zeros(2, 1, 16, 4).half()
    x, slots, i32 = torch.zeros(3, 1, 64).half(), torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int32)
    assert ops.kv_append(codes, codes, params, 4, x, x, slots) is None             # not on a GPU
    assert ops.kv_read(codes, codes, params, 4, slots, 1) is None
    assert ops.kv_attend(codes, codes, params, 4, x, i32[:, None], i32, 0.1) is None
    assert ops.kv_attend(codes, None, params, "4", x, i32[:, None], i32, 0.1) is None
    assert ops.kv_append(codes, codes) is None and ops.kv_append(codes, codes, params, 1 << 80, x, x, slots) is None
    assert ops.adapter_matmul(x[0], torch.zeros(1, 8, 64).half(), torch.zeros(1, 8, 64).half(), i32[:1], None, None, None) is None
    assert ops.adapter_matmul(1, 2, 3, 4, 5, 6, 7) is None
    with pytest.raises(TypeError):
        ops.set_operators(1)


@pytest.fixture
def python_path(monkeypatch):
    monkeypatch.setattr(_lib, "_operators", _lib._NoOperators)


def _cache(native, bits=4):
    cache = QuantizedKVCache(9, 16, 2, 128, bits=bits, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    kv = torch.randn(60, 4, 128, generator=g, device=DEV).half()
    slots = torch.randperm(9 * 16, generator=g, device=DEV)[:60]
    ops = _lib.host_operators()
    if native:
        assert ops.kv_append(*cache._cache, kv[:, :2], kv[:, 2:], slots) is True
    else:
        cache.append(kv[:, :2], kv[:, 2:], slots)
    return cache, slots


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [2, 4, 8])
def test_cache_calls_are_alike(bits, monkeypatch):
    a, slots = _cache(True, bits)
    q = torch.randn(3, 8, 256, device=DEV).half()[:, :, 64:192]
    table = torch.randint(0, 9, (3, 40), device=DEV, dtype=torch.int32)
    n = torch.tensor([9, 0, 600], device=DEV, dtype=torch.int32)
    ops = _lib.host_operators()
    native = ops.kv_attend(*a._cache, q, table, n, 128 ** -0.5), *ops.kv_read(*a._cache, slots, 2)
    assert native[0] is not None and torch.equal(a.attend(q, table, n), native[0])
    monkeypatch.setattr(_lib, "_operators", _lib._NoOperators)
    b, slots = _cache(False, bits)
    for x, y in zip(a._cache[:3], b._cache[:3]):
        assert torch.equal(x, y)
    for x, y in zip(native, (b.attend(q, table, n), *b.read(slots, dtype=torch.bfloat16))):
        assert torch.equal(x, y) and x.dtype == y.dtype and x.shape == y.shape
    b.k_codes.resize_(1, 2, 16, 16)
    with pytest.raises(RuntimeError):
        b.attend(q, table, n)
    a.k_codes.resize_(1, 2, 16, 16)
    assert ops.kv_attend(*a._cache, q, table, n, 1.0) is None


def _set(M=37, lead=None, dtype=torch.float16):
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(M, 256, generator=g, device=DEV).to(dtype)
    down = (torch.randn(3, 16, 256, generator=g, device=DEV) / 16).to(dtype)
    up = (0.1 * torch.randn(3, 16, 192, generator=g, device=DEV)).to(dtype)
    index = torch.randint(-1, 3, (M,), generator=g, device=DEV).to(torch.int32)
    return x, down, up, index, 0.5 + torch.rand(3, generator=g, device=DEV), torch.randn(M, 192, generator=g, device=DEV).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 37, 200])
def test_adapter_calls_are_alike(M, monkeypatch):
    x, down, up, index, scaling, base = _set(M)
    ops = _lib.host_operators()
    native = ops.adapter_matmul(x, down, up, index, scaling, base, None)
    assert native is not None
    spare = base.clone()
    assert ops.adapter_matmul(x, down, up, index, scaling, spare, spare) is spare and torch.equal(spare, native)
    # left to the Python path: overlaps, strides, other types, rows off a 16-byte boundary, recording into `out`
    assert ops.adapter_matmul(x, down, up, index, scaling, base, base.flatten()[8:].new_empty(0)) is None
    for bad in ((x.float(), down, up, index, scaling, base), (x[:, ::2], down, up, index, scaling, base), (x, down, up, index.long(), scaling, base),
                (x, down, up, index, scaling.half(), base), (x, down.bfloat16(), up, index, scaling, base), (x, down, up[:, :8], index, scaling, base)):
        assert ops.adapter_matmul(*bad, None) is None
    results = []
    for native_path in (True, False):
        if not native_path:
            monkeypatch.setattr(_lib, "_operators", _lib._NoOperators)
        leaves = [t.clone().requires_grad_() for t in (x, down, up, base)]
        y = adapter_matmul(leaves[0], leaves[1], leaves[2], index, scaling=scaling, base=leaves[3])
        assert ("AdapterNode" in y.grad_fn.name()) == native_path
        results.append([y.detach(), *torch.autograd.grad(y, leaves, base.flip(0))])
    assert torch.equal(results[0][0], native)
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_gradients_cannot_be_differentiated_again(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_lib, "_operators", _lib._NoOperators)
    x, down, up, index, scaling, base = _set()
    leaves = [t.requires_grad_() for t in (x, down, up)]
    grad = torch.ones_like(base, requires_grad=True)
    y = adapter_matmul(*leaves, index, scaling=scaling)
    want = torch.autograd.grad(y, leaves, grad.detach(), retain_graph=True)
    got = torch.autograd.grad(y, leaves, grad, create_graph=True)
    assert all(torch.equal(a, b.detach()) for a, b in zip(want, got))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        got[0].float().sum().backward()
    # saved tensors that are changed in place are noticed
    y = adapter_matmul(*leaves, index, scaling=scaling)
    index.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.gpu
def test_modes_and_subclasses_go_the_python_way():
    x, down, up, index, scaling, base = _set()
    want = adapter_matmul(x, down, up, index, scaling=scaling, base=base)
    ops = _lib.host_operators()

    class Sub(torch.Tensor):
        pass

    assert ops.adapter_matmul(x.as_subclass(Sub), down, up, index, scaling, base, None) is None
    assert torch.equal(adapter_matmul(x.as_subclass(Sub), down, up, index, scaling=scaling, base=base).as_subclass(torch.Tensor), want)
    with torch.inference_mode():
        assert torch.equal(adapter_matmul(x, down, up, index, scaling=scaling, base=base), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = adapter_matmul(x, down, up, index, scaling=scaling, base=base)
    side.synchronize()
    assert torch.equal(y, want) and math.isfinite(float(y.float().sum()))


@pytest.mark.gpu
def test_first_calls_may_be_captured():
    """Nothing that a first call sets up keeps it from being captured: a process whose first call of each kind is in a graph."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    program = """
import torch
from bitween_b200 import QuantizedKVCache, adapter_matmul
dev = "cuda"
g = torch.Generator(device=dev).manual_seed(0)
cache = QuantizedKVCache(700, 16, 2, 128, bits=4, device=dev)
k, v = (torch.randn(10000, 2, 128, generator=g, device=dev).half() for _ in range(2))
slots = torch.arange(10000, device=dev)
table = torch.arange(700, device=dev, dtype=torch.int32)[None].contiguous()
n = torch.tensor([9990], dtype=torch.int32, device=dev)
short = torch.tensor([300], dtype=torch.int32, device=dev)
q = torch.randn(1, 8, 128, generator=g, device=dev).half()
banks = []
for M in (20, 300):
    x = torch.randn(M, 512, generator=g, device=dev).half()
    down, up = torch.randn(2, 32, 512, generator=g, device=dev).half() / 20, torch.randn(2, 32, 256, generator=g, device=dev).half() / 20
    banks.append((x, down, up, torch.randint(-1, 2, (M,), generator=g, device=dev).int(), torch.randn(M, 256, generator=g, device=dev).half()))

def step():
    cache.append(k, v, slots)
    out = [cache.attend(q, table, n), cache.attend(q, table[:, :20], short), *cache.read(slots)]
    for x, down, up, index, grad in banks:
        leaves = [t.detach().requires_grad_() for t in (x, down, up)]
        y = adapter_matmul(*leaves, index)
        out += [y.detach(), *torch.autograd.grad(y, leaves, grad)]
    return out

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
want = step()
assert all(torch.equal(a, b) for a, b in zip(got, want)), [torch.equal(a, b) for a, b in zip(got, want)]
assert got[0].isfinite().all()
"""
    r = subprocess.run([sys.executable, "-c", program], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
