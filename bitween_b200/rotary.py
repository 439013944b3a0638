"""Rotary positions of one or several axes (time, height, width): queries and keys turned by the angles of their positions, with gradients.
No counterpart in the reference; computed by the sm_100a kernels behind bw_rotate (include/bitween_b200.h has the formula).
`QuantizedKVCache.append_rotated` rotates on the way into the cache."""
import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from .kernels import _lib

_FLOAT_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


class RotaryPositions:
    """The cosines and sines of positions 0 to max_positions - 1.

    Pair j of a head's first `rotary_dim` values, (j, j + rotary_dim/2) or where `interleaved` (2j, 2j+1), is turned by position * inv_freq[j].
    `inv_freq` defaults to base ** (-2j / rotary_dim).  With several axes of positions each pair follows one of them: `sections`, how many
    consecutive pairs each axis has, or `axes`, the axis of each pair.  `factor` multiplies cosines and sines.  Angles are computed in 64 bits; `table`, fp32
    [max_positions, rotary_dim/2, 2], holds them (cosine, sine).
    """

    def __init__(self, rotary_dim, max_positions, base=10000.0, inv_freq=None, sections=None, axes=None, interleaved=False, factor=1.0, device="cuda"):
        if rotary_dim < 2 or rotary_dim > 256 or rotary_dim % 2 != 0:
            raise ValueError("rotary_dim must be even, 2 to 256")
        if max_positions < 1:
            raise ValueError("a table needs at least one position")
        pairs = rotary_dim // 2
        if inv_freq is None:
            inv_freq = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
        inv_freq = torch.as_tensor(inv_freq, dtype=torch.float64).detach().to(device)
        if tuple(inv_freq.shape) != (pairs,):
            raise ValueError(f"inv_freq must have {pairs} frequencies")
        if sections is not None:
            if axes is not None:
                raise ValueError("give either sections or axes")
            sections = [int(n) for n in sections]
            if min(sections, default=-1) < 0 or sum(sections) != pairs:
                raise ValueError(f"sections must add up to {pairs} pairs")
            axes, self.num_axes = [a for a, n in enumerate(sections) for _ in range(n)], len(sections)
        else:
            axes = [0] * pairs if axes is None else [int(a) for a in axes]
            if len(axes) != pairs or min(axes) < 0:
                raise ValueError(f"axes must name an axis for each of {pairs} pairs")
            self.num_axes = max(axes) + 1
        if self.num_axes > 255:
            raise ValueError("at most 255 axes")
        angles = torch.arange(max_positions, dtype=torch.float64, device=inv_freq.device)[:, None] * inv_freq
        self.table = torch.stack(((angles.cos() * factor).float(), (angles.sin() * factor).float()), -1)
        self.rotary_dim, self.max_positions, self.interleaved = rotary_dim, max_positions, bool(interleaved)
        self.axes = tuple(axes)
        self.device = self.table.device
        self._shape = self.table.shape
        self._meta = (int(rotary_dim), int(self.interleaved), self.num_axes, bytes(axes), int(max_positions))

    def _checked(self, table):
        """`table` (this one's, or what came back of it for a backward pass), if the kernels can take it."""
        if table.shape != self._shape or table.dtype != torch.float32 or not table.is_contiguous() or table.device != self.device or table.data_ptr() % 16 != 0:
            raise RuntimeError("the table has been changed in shape, type or place")
        return table

    def _positions(self, positions, lead):
        """Positions for rows of the leading shape `lead`, as [tokens] or [axes, tokens]."""
        _lib.require_cuda(positions, "positions")
        if positions.dtype != torch.int64:
            raise TypeError("positions must be int64")
        if positions.device != self.device:
            raise RuntimeError(f"`positions` is on {positions.device} but the table is on {self.device}")
        if tuple(positions.shape) == tuple(lead):
            return positions.reshape(math.prod(lead)).contiguous()
        if tuple(positions.shape) != (self.num_axes, *lead):
            raise ValueError(f"positions must have shape {tuple(lead)} or {(self.num_axes, *lead)}")
        return positions.reshape(self.num_axes, math.prod(lead)).contiguous()

    def _struct(self, table, positions):
        return _lib.Rotary(self._checked(table).data_ptr(), self.max_positions, self.rotary_dim, int(self.interleaved), self.num_axes, self._meta[3],
                           positions.data_ptr(), 0 if positions.dim() == 1 else positions.shape[1])

    def rotate(self, positions, *xs):
        """One or two tensors [..., heads, dim] (queries, and keys with heads of their own; fp32, fp16 or bf16; dim at least rotary_dim) rotated, in
        one launch.  Returns new tensors, rounded once: one for one, a tuple for two.  `positions`, int64: of the tensors' leading shape, or
        with several axes [axes, *leading shape].  A position outside the table gives NaN.  Values behind the first rotary_dim are copied.  Differentiable."""
        ops = _lib._operators or _lib.host_operators()
        out = ops.rotate(self.table, self._meta, positions, *xs)
        if out is not None:
            return out
        _lib.refuse_recorders("rotate")
        if not torch.jit.is_tracing():
            at, *rows = self._arguments(positions, xs)
            out = ops.rotate(self._checked(self.table), self._meta, at, *rows)
        if out is not None:
            out = tuple(y.view(x.shape) for x, y in zip(xs, (out,) if len(xs) == 1 else out))
        elif _lib.for_autograd(*xs):
            out = RotateFunction.apply(self, positions, *xs)
        else:
            out = _rotate(self, self.table, at, rows, [x.shape for x in xs], False)
        return out[0] if len(xs) == 1 else tuple(out)

    def _arguments(self, positions, xs):
        """(positions, tensors...) of a call, checked, as the kernels take them."""
        if not 1 <= len(xs) <= 2:
            raise ValueError("rotate takes one or two tensors")
        for x in xs:
            _lib.require_cuda(x, "x")
            if x.dtype not in _FLOAT_DTYPES or x.dtype != xs[0].dtype:
                raise TypeError("the tensors to rotate must have one dtype: float32, float16 or bfloat16")
            if x.device != self.device:
                raise RuntimeError(f"`x` is on {x.device} but the table is on {self.device}")
            if x.dim() < 2 or x.shape[:-2] != xs[0].shape[:-2] or x.shape[-1] != xs[0].shape[-1] or x.shape[-1] < self.rotary_dim:
                raise ValueError(f"the tensors to rotate must be [..., heads, dim] of one leading shape and one dim of at least {self.rotary_dim}")
        return self._positions(positions, xs[0].shape[:-2]), *(_rows(x) for x in xs)

    def __repr__(self):
        return f"RotaryPositions(rotary_dim={self.rotary_dim}, max_positions={self.max_positions}, num_axes={self.num_axes}, interleaved={self.interleaved})"


def _rows(x):
    """x [..., heads, dim] as [tokens, heads, dim] whose values lie side by side."""
    x = x.resolve_neg()
    x = x.reshape(math.prod(x.shape[:-2]), *x.shape[-2:]) if x.dim() != 3 else x
    return x if x.stride(2) == 1 else x.contiguous()


def _rotate(rotary, table, positions, rows, shapes, inverse):
    """New tensors of `shapes`: those of `rows` ([tokens, heads, dim], as `_rows` gives them) that are there, turned (or turned back).  None where there is none."""
    outs = [None if x is None else torch.empty(shape, dtype=x.dtype, device=x.device) for x, shape in zip(rows, shapes)]
    given = [(x, out) for x, out in zip(rows, outs) if out is not None and out.numel()]
    if given:
        args = []
        for x, out in given:
            args += [x.data_ptr(), x.shape[1], x.stride(0), x.stride(1), out.data_ptr()]
        args += [None, 0, 0, 0, None] * (2 - len(given))
        x = given[0][0]
        L = _lib.lib()
        with _lib.on_device(rotary.device):
            rc = L.bw_rotate(ctypes.byref(rotary._struct(table, positions)), x.shape[0], x.shape[2], _lib.dtype_code(x.dtype), int(inverse), *args,
                             _lib.raw_stream(rotary.device))
        _lib.check(rc)
    return outs


class RotateFunction(torch.autograd.Function):
    """apply(rotary, positions, *xs): what `rotate` says, of tensors that it may have checked or not (a traced call runs again with others)."""

    @staticmethod
    def forward(ctx, rotary, positions, *xs):
        positions, *rows = rotary._arguments(positions, xs)
        ctx.rotary = rotary
        ctx.save_for_backward(rotary.table, positions)
        ctx.like = (positions.shape, positions.dtype, positions.device)
        ctx.set_materialize_grads(False)
        return tuple(_rotate(rotary, rotary.table, positions, rows, [x.shape for x in xs], False))

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        _lib.refuse_capture("rotate")
        table, positions = ctx.saved_tensors
        # (hooks may have made other tensors of them in the meantime: moved, packed)
        if (positions.shape, positions.dtype, positions.device) != ctx.like:
            raise RuntimeError("rotate: a tensor saved for the backward pass has come back from its hooks in another shape, type or place")
        wanted = [_rows(g) if g is not None and need else None for g, need in zip(grads, ctx.needs_input_grad[2:])]
        return (None, None, *_rotate(ctx.rotary, table, positions.contiguous(), wanted, [None if g is None else g.shape for g in grads], True))
