"""Low-rank adapters of many requests beside a shared projection: each row of a batch has an adapter of its own, or none, and all
rows go through one QuantizedLinear.  (The reference wraps one adapter around one linear, bitween/utils/singlora.py; here the
adapters of a layer are one bank.)  Computed by the sm_100a kernels behind bw_adapter_forward and bw_adapter_backward."""
import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .kernels import _lib
from .modules import QuantizedLinear

_DTYPES = (torch.float16, torch.bfloat16)


def _aligned(t):
    """`t` contiguous and on a 16-byte boundary."""
    t = t if t.is_contiguous() else t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _forward(x, down, up, index, scaling, base, out, keep):
    """(out [M, N], hidden): `hidden` is what the backward pass needs again, or None."""
    M, K = x.shape
    adapters, rank, N = up.shape
    dev = x.device
    if out is None:
        out = torch.empty((M, N), dtype=x.dtype, device=dev)
    L = _lib.lib()
    with _lib.on_device(dev):
        need = L.bw_adapter_hidden_bytes(M, rank)
        hidden = torch.empty(need, dtype=torch.uint8, device=dev) if keep else _lib.workspace(dev, need)
        rc = L.bw_adapter_forward(x.data_ptr(), _lib.dtype_code(x.dtype), M, N, K, down.data_ptr(), up.data_ptr(), adapters, rank, index.data_ptr(),
                                  None if scaling is None else scaling.data_ptr(), None if base is None else base.data_ptr(), out.data_ptr(),
                                  None if hidden is None else hidden.data_ptr(), 0 if hidden is None else hidden.numel(), _lib.raw_stream(dev))
    _lib.check(rc)
    return out, hidden if keep else None


def _arguments(x, down, up, index, scaling, base, out=None):
    """(x [M, K], down, up, index [M], scaling, base [M, N]) of a call, checked, as the kernels take them."""
    _lib.require_cuda(x, "x")
    if x.dtype not in _DTYPES:
        raise TypeError(f"adapter_matmul: unsupported dtype {x.dtype} (float16/bfloat16)")
    if down.dim() != 3 or up.dim() != 3 or down.shape[:2] != up.shape[:2]:
        raise ValueError("down and up must be [adapters, rank, in_features] and [adapters, rank, out_features]")
    adapters, rank, K = down.shape
    N = up.shape[2]
    if adapters < 1 or not 1 <= rank <= 256 or K < 1 or N < 1:
        raise ValueError("a bank holds at least one adapter, of rank 1 to 256")
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"x has {x.shape[-1] if x.dim() else 0} input features but down has {K}")
    lead = x.shape[:-1]
    if index.dtype != torch.int32:
        raise TypeError("index must be int32")
    x2 = x.reshape(-1, K)
    M = x2.shape[0]
    if index.numel() != M or (index.dim() != 1 and index.shape != lead):
        raise ValueError(f"index must name an adapter for each of the {M} rows of x")
    if base is not None and base.shape != (*lead, N):
        raise ValueError(f"base must have shape {(*lead, N)}")
    if scaling is not None:
        if scaling.dtype != torch.float32 or tuple(scaling.shape) != (adapters,):
            raise ValueError(f"scaling must be fp32 [{adapters}]")
        if scaling.requires_grad:
            raise ValueError("scaling has no gradient; detach it")
    for name, t in (("down", down), ("up", up), ("index", index), ("scaling", scaling), ("base", base), ("out", out)):
        if t is None:
            continue
        if t.device != x.device:
            raise RuntimeError(f"`{name}` is on {t.device} but x is on {x.device}")
        if name in ("down", "up", "base", "out") and t.dtype != x.dtype:
            raise TypeError(f"`{name}` is {t.dtype} but x is {x.dtype}")
    index = index.reshape(-1).contiguous()
    if scaling is not None:
        scaling = scaling.contiguous()
    base2 = None if base is None else _aligned(base.reshape(M, N))
    return _aligned(x2), _aligned(down), _aligned(up), index, scaling, base2


class AdapterFunction(torch.autograd.Function):
    """apply(x, down, up, index, scaling, base): what `adapter_matmul` says, of arguments that it may have checked or not (a traced call runs again with other tensors)."""

    @staticmethod
    def forward(ctx, x, down, up, index, scaling, base):
        ctx.shape = x.shape
        x, down, up, index, scaling, base = _arguments(x, down, up, index, scaling, base)
        out = torch.empty((*ctx.shape[:-1], up.shape[2]), dtype=x.dtype, device=x.device)
        _, hidden = _forward(x, down, up, index, scaling, base, out, ctx.needs_input_grad[2])
        ctx.save_for_backward(x, down, up, index, scaling, hidden)
        ctx.like = [None if t is None else (t.shape, t.dtype, t.device) for t in (x, down, up, index, scaling, hidden)]
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        saved = ctx.saved_tensors
        # (hooks may have made other tensors of them in the meantime: moved, packed)
        if any((t is None) != (like is None) or (t is not None and (t.shape, t.dtype, t.device) != like) for t, like in zip(saved, ctx.like)):
            raise RuntimeError("adapter_matmul: a tensor saved for the backward pass has come back from its hooks in another shape, type or place")
        x, down, up, index, scaling, hidden = (t if t is None else _aligned(t.resolve_neg()) for t in saved)
        want_x, want_down, want_up = ctx.needs_input_grad[:3]
        grads = [torch.empty_like(t) if want else None for t, want in ((x, want_x), (down, want_down), (up, want_up))]
        if want_x or want_down or want_up:
            M, K = x.shape
            adapters, rank, N = up.shape
            dev = x.device
            g = _aligned(grad_out)
            L = _lib.lib()
            with _lib.on_device(dev):
                ws = _lib.workspace(dev, L.bw_adapter_hidden_bytes(M, rank))
                rc = L.bw_adapter_backward(g.data_ptr(), _lib.dtype_code(x.dtype), x.data_ptr(), M, N, K, down.data_ptr(), up.data_ptr(), adapters, rank,
                                           index.data_ptr(), None if scaling is None else scaling.data_ptr(),
                                           None if hidden is None else hidden.data_ptr(), 0 if hidden is None else hidden.numel(),
                                           *(None if t is None else t.data_ptr() for t in grads),
                                           None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), _lib.raw_stream(dev))
            _lib.check(rc)
        if want_x:
            grads[0] = grads[0].view(ctx.shape)
        return (*grads, None, None, grad_out if ctx.needs_input_grad[5] else None)


def adapter_matmul(x, down, up, index, scaling=None, base=None, out=None):
    """base[t] + scaling[i] * up[i]^T (down[i] x[t]) with i = index[t], for x [..., K] and the bank `down` [adapters, rank, K], `up`
    [adapters, rank, N] (both rank-major: `up` is the transpose of a PEFT checkpoint's lora_B).  Returns [..., N].

    `index`, int32 of x's leading shape (or flat): the adapter of each row; rows below 0 have none and get `base` (zeros without
    one); an index beyond the bank gives NaN.  `scaling`: fp32 [adapters] or None (ones); it has no gradient.  x, down, up and base share one
    dtype, fp16 or bf16; sums are fp32 and the result is rounded once.  Ranks up to 256.  Differentiable in x, down, up and base.
    `out`, a contiguous tensor of the result's shape, takes the result where no gradient is recorded (one that requires a gradient is refused, too, and so is any tensor with a
    forward-mode tangent); it may be `base` itself."""
    y = (_lib._operators or _lib.host_operators()).adapter_matmul(x, down, up, index, scaling, base, out)
    if y is not None:
        return y
    _lib.refuse_recorders("adapter_matmul", traced=out is not None)
    if out is None and _lib.for_autograd(x, down, up, scaling, base):
        return AdapterFunction.apply(x, down, up, index, scaling, base)
    args = _arguments(x, down, up, index, scaling, base, out)
    lead, (M, N) = x.shape[:-1], (args[0].shape[0], up.shape[2])
    if out is None:
        return _forward(*args, None, False)[0].view(*lead, N)
    if _lib.for_autograd(x, down, up, scaling, base, out):
        raise ValueError("`out` is for calls that record no gradient and have no forward-mode tangent")
    if out.shape != (*lead, N) or not out.is_contiguous():
        raise ValueError(f"`out` must be contiguous {(*lead, N)}")
    if out.data_ptr() % 16 != 0:
        return out.copy_(_forward(*args, None, False)[0].view(*lead, N))
    for i in range(6):          # kernels store outputs while others still read
        t = args[i]
        if t is not None and t.data_ptr() < out.data_ptr() + out.nbytes and out.data_ptr() < t.data_ptr() + t.nbytes and \
                not (i == 5 and t.data_ptr() == out.data_ptr()):
            args = (*args[:i], t.clone(), *args[i + 1:])
    _forward(*args, out.view(M, N), False)
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)      # (written in place, as autograd has to know)
    return out


class AdaptedLinear(nn.Module):
    """A QuantizedLinear and a bank of low-rank adapters beside it: forward(x, index) is layer(x) plus each row's adapter.  (The layer is called as a module, with
    its hooks; one whose class has a forward of its own, too.)

    The packed layer stays as it is (frozen, shared); `down` [adapters, rank, in_features] and `up` [adapters, rank, out_features] are
    parameters of `dtype` (fp16 or bf16), in which x is taken and the result is returned.  `scaling` is a buffer, [adapters].  New adapters
    have `up` zero, so that they change nothing."""

    def __init__(self, layer, num_adapters, rank, scaling=1.0, dtype=torch.float16):
        super().__init__()
        if not isinstance(layer, QuantizedLinear):
            raise TypeError("AdaptedLinear wraps a QuantizedLinear")
        if dtype not in _DTYPES:
            raise TypeError(f"unsupported dtype {dtype} (float16/bfloat16)")
        if num_adapters < 1 or not 1 <= rank <= 256:
            raise ValueError("a bank holds at least one adapter, of rank 1 to 256")
        device = layer.qweight.device
        self.layer = layer
        self.down = nn.Parameter((torch.randn((num_adapters, rank, layer.in_features), device=device) * layer.in_features ** -0.5).to(dtype))
        self.up = nn.Parameter(torch.zeros((num_adapters, rank, layer.out_features), dtype=dtype, device=device))
        self.register_buffer("scaling", torch.full((num_adapters,), float(scaling), device=device))

    def forward(self, x, index):
        layer, dtype = self.layer, self.down.dtype
        x = x.to(dtype)
        if type(layer).forward is QuantizedLinear.forward and "forward" not in layer.__dict__:
            base = layer(x, out_dtype=dtype)
            # (what a hook has seen, or given, is not written over)
            in_place = not (layer._forward_hooks or nn.modules.module._global_forward_hooks)
        else:                                      # a layer with a forward of its own
            base, in_place = layer(x), False
        base = base.to(dtype)
        in_place = in_place and not (torch.is_grad_enabled() and (base.requires_grad or self.down.requires_grad or self.up.requires_grad))
        scaling = self.scaling.float()
        y = (_lib._operators or _lib.host_operators()).adapter_matmul(x, self.down, self.up, index, scaling, base, base if in_place else None)
        if y is not None:
            return y
        # (a traced call, and one with a tangent, is the autograd function's)
        in_place = in_place and not torch.jit.is_tracing() and not _lib.any_tangent(x, self.down, self.up)
        return adapter_matmul(x, self.down, self.up, index, scaling=scaling, base=base, out=base if in_place else None)

    def extra_repr(self):
        return f"num_adapters={self.down.shape[0]}, rank={self.down.shape[1]}"
