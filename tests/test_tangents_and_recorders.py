"""Calls of the operators beside the linears with a forward-mode tangent, and under what writes torch operations down to run them again: their kernels are no torch
operations, so that such a call is a node of its own, or refused, and never an empty output without a word."""
import contextlib

import pytest
import torch
import torch.autograd.forward_ad as fwad
from torch.fx.experimental.proxy_tensor import make_fx

from bitween_b200 import AdaptedLinear, QuantizedKVCache, QuantizedLinear, RotaryPositions, adapter_matmul, token_log_probs
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


def test_token_log_probs(library):
    t, x, column = torch.arange(3), torch.randn(3, 50), torch.arange(3)[:, None]
    for call in (lambda x: token_log_probs(x, t).log_probs, lambda x: token_log_probs(x, entropy=True).entropy, lambda x: tuple(token_log_probs(x, t, entropy=True, top=3)),
                 lambda x: token_log_probs(x[:, :40].unflatten(0, (3, 1)), column, top=2).top_log_probs):
        _tangent_refused(call, x)
        _not_recorded(call, x)
        traced = _traced(call, x)
        assert "^TokenLogProbsFunction" in str(traced.graph) and "aten::empty" not in str(traced.graph)
        library.calls.clear()
        traced(x)
        assert library.calls == ["bw_token_log_probs"]
    traced = _traced(lambda x, t: token_log_probs(x, t, top=3).log_probs, (x, t))
    library.calls.clear()
    for bad in ((x.double(), t), (x, t.int()), (x, t[:2]), (x[:, :2], t)):
        with pytest.raises(Exception, match="must|unsupported"):
            traced(*bad)
    assert not library.calls
    assert token_log_probs(x) == (None,) * 4


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_traced_log_probs_run_again_on_other_tensors():
    g = torch.Generator(device="cuda").manual_seed(2)
    x, other = (torch.randn(4, 7, 1003, generator=g, device="cuda").bfloat16() for _ in range(2))
    t = torch.randint(-1, 1003, (4, 7), generator=g, device="cuda")
    traced = torch.jit.trace(lambda x, t: tuple(token_log_probs(x, t, entropy=True, top=4)), (x, t), check_trace=False)
    columns = torch.randn(1003, 7, 4, generator=g, device="cuda").bfloat16().permute(2, 1, 0)
    for a in (x, other, columns, torch.cat((x, other), 1)[:, 3:10]):
        for at in (t, t.flip(0)):
            assert all(torch.equal(got, want) for got, want in zip(traced(a, at), token_log_probs(a, at, entropy=True, top=4)))
    leaf = other.clone().requires_grad_()
    ones = torch.ones(4, 7, device="cuda")
    (got,) = torch.autograd.grad(traced(leaf, t)[0], leaf, ones)
    (want,) = torch.autograd.grad(token_log_probs(leaf, t).log_probs, leaf, ones)
    assert torch.equal(got, want)
    with fwad.dual_level(), pytest.raises(NotImplementedError):
        token_log_probs(fwad.make_dual(x, x), t)
    _not_recorded(lambda x: token_log_probs(x, t).log_probs, x)


@pytest.mark.gpu
def test_gradients_of_rows_with_two_strides_on_both_paths(monkeypatch):
    """Rows whose leading dimensions are not one stride, and outputs that are written in place."""
    g = torch.Generator(device="cuda").manual_seed(3)
    big, t = torch.randn(4, 9, 1003, generator=g, device="cuda"), torch.randint(0, 1003, (4, 8), generator=g, device="cuda")
    results = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(_lib, "_operators", _lib._NoOperators)
        leaf = big.clone().requires_grad_()
        r = token_log_probs(leaf[:, :-1], t, entropy=True, top=2)
        r.log_probs.mul_(0.5)
        (r.log_probs.sum() + r.entropy.sum() + r.top_log_probs[..., 1].sum()).backward()
        results.append((*(y.detach() for y in r), leaf.grad))
    assert all(torch.equal(a, b) for a, b in zip(*results)) and not bool(results[0][-1][:, -1].any())
    p = torch.softmax(big[:, :-1].double(), -1)
    inner = p.log() + torch.special.entr(p).sum(-1, keepdim=True)
    want = p * (-1.5 - inner)
    want.scatter_add_(-1, t[..., None], torch.full((4, 8, 1), 0.5, dtype=torch.float64, device="cuda"))
    want.scatter_add_(-1, results[0][3][..., 1:], torch.ones(4, 8, 1, dtype=torch.float64, device="cuda"))
    # exponents of spans of less than 16 good to 2^-18, relative, of p (1.5 + |inner| + H); an entry of a token is a sum of up to three parts
    size = p * (1.5 + inner.abs() + 7)
    assert bool(((results[0][-1][:, :-1].double() - want).abs() <= 2.0 ** -18 * size + 2.0 ** -21 * (want.abs() + size)).all())


def _cache_calls(dev):
    """Calls of a cache whose codes have no derivative: (call, its float tensor or slots, whether a tangent of that is refused)."""
    cache, r, p = QuantizedKVCache(4, 16, 2, 64, bits=4, device=dev), RotaryPositions(64, 50, device=dev), torch.arange(3, device=dev)
    x, table, n = torch.randn(3, 2, 64, device=dev).half(), torch.zeros(3, 1, dtype=torch.int32, device=dev), torch.ones(3, dtype=torch.int32, device=dev)
    return [(lambda q: cache.attend(q, table, n), x, True), (lambda q: cache.attend(q, table, n, window=3), x, True),
            (lambda q: cache.append_rotated(q, x, x, p, r, p), x, True), (lambda k: cache.append_rotated(None, k, k, p, r, p), x, False),
            (lambda k: cache.append(k, k, p), x, False), (lambda s: cache.read(s), p, False)]


def _cache_refusals(dev):
    for call, x, derived in _cache_calls(dev):
        _not_recorded(call, x)
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            torch.jit.trace(call, x, check_trace=False)
        if derived:
            with pytest.raises(ValueError, match="no gradient"):
                call(x.clone().requires_grad_())
        for mode in (contextlib.nullcontext, torch.no_grad) if derived else ():
            with fwad.dual_level(), mode():
                dual = fwad.make_dual(x, torch.ones_like(x))
                with pytest.raises(ValueError, match="no forward-mode derivative"):
                    call(dual)
                call(dual.detach())


def test_the_cache(library):
    _cache_refusals("cpu")
    assert "bw_kv_attend" in library.calls and "bw_kv_attend_window" in library.calls and "bw_kv_append_rotated" in library.calls


@pytest.mark.gpu
def test_the_cache_on_the_gpu():
    _cache_refusals("cuda")


def test_adapter_matmul(library):
    x, down, up, index = torch.randn(3, 64).half(), torch.randn(2, 8, 64).half(), torch.randn(2, 8, 32).half(), torch.zeros(3, dtype=torch.int32)
    base = torch.zeros(3, 32).half()
    lead, lead_base = index[:, None], base[:, None]
    for call, arg in ((lambda x: adapter_matmul(x, down, up, index), x), (lambda u: adapter_matmul(x, down, u, index, base=base), up),
                      (lambda x: adapter_matmul(x[:, None], down, up, lead, base=lead_base), x)):
        _tangent_refused(call, arg)
        _not_recorded(call, arg)
        traced = _traced(call, arg)
        assert "^AdapterFunction" in str(traced.graph) and "aten::empty" not in str(traced.graph)
        library.calls.clear()
        traced(arg)
        assert library.calls == ["bw_adapter_hidden_bytes", "bw_adapter_forward"]
    out = torch.empty(3, 32).half()
    with torch.no_grad():
        _not_recorded(lambda x: adapter_matmul(x, down, up, index, out=out), x)
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            torch.jit.trace(lambda x: adapter_matmul(x, down, up, index, out=out), x, check_trace=False)
        with fwad.dual_level():
            for kw in ({"x": fwad.make_dual(x, x)}, {"up": fwad.make_dual(up, up)}, {"base": fwad.make_dual(base, base)}):
                with pytest.raises(ValueError, match="forward-mode"):
                    adapter_matmul(**({"x": x, "down": down, "up": up, "index": index, "out": out} | kw))


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_traced_adapters_run_again_on_other_tensors(monkeypatch):
    g = torch.Generator(device="cuda").manual_seed(4)
    layer = AdaptedLinear(QuantizedLinear.from_float(torch.nn.Linear(128, 96).cuda().half(), bits=4, group_size=64), 2, 8)
    with torch.no_grad():
        layer.up.copy_(torch.randn(layer.up.shape, generator=g, device="cuda"))
    x, other = (torch.randn(2, 3, 128, generator=g, device="cuda").half() for _ in range(2))
    index, turned = torch.tensor([[0, 1, -1], [1, 1, 0]], dtype=torch.int32, device="cuda"), torch.randn(128, 3, 2, generator=g, device="cuda").half().permute(2, 1, 0)
    for mode in (torch.no_grad, torch.enable_grad):
        with mode():
            traced = torch.jit.trace(layer, (x, index), check_trace=False)
            for a in (x, other, turned):
                for i in (index, index.flip(0)):
                    assert torch.equal(traced(a, i), layer(a, i))
            with fwad.dual_level(), pytest.raises(NotImplementedError):
                layer(fwad.make_dual(x, x), index)
    down, up = (t.detach() for t in (layer.down, layer.up))
    results = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(_lib, "_operators", _lib._NoOperators)
        leaf, bank = turned.clone().requires_grad_(), up.clone().requires_grad_()
        y = adapter_matmul(leaf, down, bank, index)
        y.mul_(0.5)
        results.append((y.detach(), *torch.autograd.grad(y, (leaf, bank), torch.ones_like(y))))
    assert all(torch.equal(a, b) for a, b in zip(*results)) and results[0][1].shape == (2, 3, 128)


@pytest.mark.gpu
def test_modes_that_only_look_on_change_nothing():
    """Dispatch modes of a program's own (counters, loggers) see the outputs' allocations and are no recorders."""
    from torch.utils._python_dispatch import TorchDispatchMode
    from torch.utils.flop_counter import FlopCounterMode

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    g = torch.Generator(device="cuda").manual_seed(5)
    r, p = RotaryPositions(64, 50), torch.arange(3, device="cuda")
    x, logits = torch.randn(3, 2, 64, generator=g, device="cuda").half(), torch.randn(3, 50, generator=g, device="cuda")
    down, up, index = torch.randn(2, 8, 64, generator=g, device="cuda").half(), torch.randn(2, 8, 32, generator=g, device="cuda").half(), torch.tensor([0, -1, 1], dtype=torch.int32, device="cuda")
    cache, table, n = QuantizedKVCache(4, 16, 2, 64, bits=4), torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.full((3,), 3, dtype=torch.int32, device="cuda")

    def step():
        cache.append(x, x, p)
        q = cache.append_rotated(x, x, x, p, r, p)
        leaf = x.clone().requires_grad_()
        y = r.rotate(p, leaf)
        return [q, *cache.read(p), cache.attend(q, table, n, window=2), cache.attend(q, table, n), r.rotate(p, x), *token_log_probs(logits, p, entropy=True, top=2),
                adapter_matmul(x[:, 0], down, up, index), adapter_matmul(x[:, 0], down, up, index, out=torch.empty(3, 32, device="cuda").half()), *torch.autograd.grad(y, leaf, x)]

    want = step()
    for mode in (Mode, lambda: FlopCounterMode(display=False), lambda: torch.device("cuda")):
        with mode():
            got = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
