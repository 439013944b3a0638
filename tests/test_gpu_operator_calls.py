"""Calls of the cache and the adapters that the documentation allows and that are easily got wrong."""
import pytest
import torch

from bitween_b200 import adapter_matmul
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
