"""Calls of the cache and the adapters that the documentation allows and that are easily got wrong."""
import pytest
import torch

from bitween_b200 import AdaptedLinear, QuantizedLinear, adapter_matmul
from bitween_b200.kernels import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _bank(M, K, N, n, r, dtype=torch.float16, seed=1):
    g = _gen(seed)
    x, down, up = torch.randn(M, K, generator=g, device=DEV), torch.randn(n, r, K, generator=g, device=DEV) * K ** -0.5, 0.2 * torch.randn(n, r, N, generator=g, device=DEV)
    return (*(t.to(dtype) for t in (x, down, up)), torch.randint(-1, n, (M,), generator=g, device=DEV).to(torch.int32), torch.randn(M, N, generator=g, device=DEV).to(dtype))


@pytest.mark.parametrize("n,r", [(4, 8), (8, 16), (40, 64)])
def test_one_tensor_as_several_arguments_and_as_the_result(n, r):
    """A tensor that is base and result may be another argument as well: what is read of that is what stood there before."""
    K = N = 128
    x, down, up, index, _ = _bank(n * r, K, N, n, r)
    ops, lead = _lib.host_operators(), (n, r)
    for which in ("up", "down", "x"):
        args = {"x": x.view(*lead, K), "down": down.clone(), "up": up.clone()}
        both = args[which]
        want = adapter_matmul(args["x"], args["down"], args["up"], index.view(lead), base=both.clone())
        assert ops.adapter_matmul(args["x"], args["down"], args["up"], index.view(lead), None, both, both) is None
        got = adapter_matmul(args["x"], args["down"], args["up"], index.view(lead), base=both, out=both)
        assert got is both and torch.equal(got, want)


@pytest.mark.parametrize("native", [True, False])
def test_a_result_that_requires_a_gradient_is_refused(native, monkeypatch):
    """Written in place it would keep the history of what stood there before."""
    if not native:
        monkeypatch.setattr(_lib, "_operators", _lib._NoOperators)
    x, down, up, index, base = _bank(9, 64, 128, 2, 8)
    for out in (base.clone().requires_grad_(), base.clone().requires_grad_() * 2):
        before = out.detach().clone()
        with pytest.raises(ValueError, match="no gradient"):
            adapter_matmul(x, down, up, index, base=base, out=out)
        assert torch.equal(out.detach(), before)
        with torch.no_grad():
            adapter_matmul(x, down, up, index, base=base, out=out)
        assert torch.equal(out.detach(), adapter_matmul(x, down, up, index, base=base))


def _spread(t):
    """The same values, not contiguous."""
    wide = t.new_empty((*t.shape, 2))
    wide[..., 0] = t
    return wide[..., 0]


def _shifted(t):
    """The same values, off a 16-byte boundary."""
    return torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)


@pytest.mark.parametrize("native", [True, False])
def test_saved_tensors_that_hooks_have_moved_or_packed(native, monkeypatch):
    """What the hooks give back is what the backward pass works on: in any layout, but of the saved shape, type and device."""
    if not native:
        monkeypatch.setattr(_lib, "_operators", _lib._NoOperators)
    x, down, up, index, base = _bank(40, 64, 128, 2, 8)
    scaling = torch.tensor([0.5, 2.0], device=DEV)

    def gradients(hooks=None):
        leaves = [t.clone().requires_grad_() for t in (x, down, up)]
        if hooks is None:
            y = adapter_matmul(*leaves, index, scaling=scaling)
        else:
            with hooks:
                y = adapter_matmul(*leaves, index, scaling=scaling)
        assert ("AdapterNode" in y.grad_fn.name()) == native
        return torch.autograd.grad(y, leaves, base)

    want = gradients()
    hooks = torch.autograd.graph.saved_tensors_hooks
    for same in (torch.autograd.graph.save_on_cpu(), hooks(lambda t: t.clone(), _spread), hooks(lambda t: t.clone(), _shifted), hooks(lambda t: t.cpu(), lambda t: t.to(DEV))):
        assert all(torch.equal(a, b) for a, b in zip(gradients(same), want))
    for other in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t.flatten(), lambda t: t[:1], lambda t: t.bfloat16() if t.dtype == torch.float16 else t):
        with pytest.raises(RuntimeError, match="come back from its hooks"):
            gradients(hooks(lambda t: t.clone(), other))


def _adapted(dtype, layer_class=QuantizedLinear):
    lin = torch.nn.Linear(128, 256, bias=True).to(DEV)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(256, 128, generator=_gen(5), device=DEV) * 0.05)
        lin.bias.copy_(torch.randn(256, generator=_gen(6), device=DEV) * 0.05)
    adapted = AdaptedLinear(layer_class.from_float(lin, bits=4, group_size=64), 2, 8, dtype=dtype)
    with torch.no_grad():
        adapted.down.copy_(torch.randn(adapted.down.shape, generator=_gen(7), device=DEV) * 0.1)
        adapted.up.copy_(torch.randn(adapted.up.shape, generator=_gen(8), device=DEV) * 0.1)
    return adapted, torch.randn(5, 128, generator=_gen(9), device=DEV).to(dtype), torch.tensor([0, 1, -1, 0, 1], dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("recording", [True, False])
def test_adapted_linear_calls_its_layer(dtype, recording):
    """Hooks of the wrapped layer see its input and output, may change the output, and what they keep stays as it was."""
    adapted, x, index = _adapted(dtype)
    seen = []
    with torch.set_grad_enabled(recording):
        want = adapted(x, index).detach()
        base = adapted.layer(x, out_dtype=dtype).detach()
        pre = adapted.layer.register_forward_pre_hook(lambda m, args: seen.append(args[0]))
        post = adapted.layer.register_forward_hook(lambda m, args, out: seen.append(out))
        assert torch.equal(adapted(x, index).detach(), want)
        assert len(seen) == 2 and torch.equal(seen[0], x) and torch.equal(seen[1].detach(), base)
        pre.remove()
        post.remove()
        twice = adapted.layer.register_forward_hook(lambda m, args, out: out * 2)
        doubled = adapted(x, index).detach()
        twice.remove()
        assert torch.equal(doubled, adapter_matmul(x, adapted.down.detach(), adapted.up.detach(), index, scaling=adapted.scaling, base=base * 2))
        adapted.layer.out_dtype = torch.float32                       # (the layer's own setting is for its own callers)
        assert torch.equal(adapted(x, index).detach(), want) and want.dtype == dtype


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_adapted_linear_with_a_layer_that_has_a_forward_of_its_own(dtype):
    class Halved(QuantizedLinear):
        def forward(self, x):
            return super().forward(x) * 0.5

    adapted, x, index = _adapted(dtype, Halved)
    with torch.no_grad():
        got = adapted(x, index)
        assert torch.equal(got, adapter_matmul(x, adapted.down, adapted.up, index, scaling=adapted.scaling, base=adapted.layer(x).to(dtype)))
        adapted.layer.forward = lambda x: torch.zeros(*x.shape[:-1], 256, dtype=dtype, device=DEV)
        assert torch.equal(adapted(x, index), adapter_matmul(x, adapted.down, adapted.up, index, scaling=adapted.scaling))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_adapted_linear_takes_the_native_way_where_nothing_is_recorded(dtype, monkeypatch):
    adapted, x, index = _adapted(dtype)
    with torch.no_grad():
        want = adapted(x, index)
        monkeypatch.setattr("bitween_b200.modules.QuantizedLinearFunction.apply", None)
        assert torch.equal(adapted(x, index), want)


def test_tensor_memory_is_shared_with_the_packed_linears_on_other_streams():
    """Kernels that take an SM's whole tensor memory (many tokens beside adapters), in clusters and not, captured and replayed beside packed linears of all sizes."""
    lin = torch.nn.Linear(1024, 2048).to(DEV).half()
    layer = QuantizedLinear.from_float(lin, bits=4, group_size=128)
    with torch.no_grad():
        tokens = [torch.randn(m, 1024, generator=_gen(70 + m), device=DEV).half() for m in (33, 64, 200, 600, 2100)]
        for t in tokens:
            layer(t)
    banks = [_bank(m, 1024, 2048, 2, 64, dtype, seed=80 + m) for m, dtype in ((2100, torch.float16), (2300, torch.bfloat16))]

    def step(i):
        if i == 2:
            with torch.no_grad():
                return [layer(t) for t in tokens]
        x, down, up, index, base = banks[i]
        leaves = [t.detach().requires_grad_() for t in (x, down, up)]
        y = adapter_matmul(*leaves, index.sort().values, base=base)
        return [y.detach(), *torch.autograd.grad(y, leaves, base)]

    want = [step(i) for i in range(3)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(3):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(i)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(i))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, ref))
    assert _lib.lib().bw_device_status() == 0
