"""A paged key-value cache quantised as it is written: 2, 4 or 8 bits, one scale and zero point per token and head, by the
rounding of quantize_rtn.  No counterpart in the reference; computed by the sm_100a kernels behind bw_kv_append, bw_kv_read and
bw_kv_attend (include/bitween_b200.h has the format)."""
import ctypes
import math
import operator

import torch

from .kernels import _lib
from .rotary import RotaryPositions

_FLOAT_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _refuse_derivatives(name, q):
    if q.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} has no gradient; detach q or call it under torch.no_grad()")
    if _lib.any_tangent(q):
        raise ValueError(f"{name} has no forward-mode derivative; detach q")


class QuantizedKVCache:
    """`num_pages` pages of `page_size` tokens; slot s is row s % page_size of page s // page_size.

    `k_codes`, `v_codes` int32 [pages, heads, page_size, head_dim * bits / 32], packed like weights, and `params` fp16
    [pages, heads, page_size, 4]: scale and zero point of the key, then of the value.  A row stands for scale * (code - zero_point).
    Which pages belong to which sequence is the caller's: `append` and `read` take slots, `attend` a table of pages.
    """

    def __init__(self, num_pages, page_size, num_kv_heads, head_dim, bits=8, device="cuda"):
        if bits not in (2, 4, 8):
            raise ValueError("Only 2, 4, or 8 bits are supported.")
        if num_pages < 0 or page_size < 1 or num_kv_heads < 1:
            raise ValueError("a cache needs at least one head and pages of at least one token")
        if head_dim < 1 or head_dim > 256 or head_dim % (32 // bits) != 0:
            raise ValueError(f"head_dim must be a multiple of {32 // bits} codes per int32, at most 256")
        rows = (num_pages, num_kv_heads, page_size)
        words = head_dim * bits // 32
        self._set_up(torch.zeros((*rows, words), dtype=torch.int32, device=device), torch.zeros((*rows, words), dtype=torch.int32, device=device),
                     torch.zeros((*rows, 4), dtype=torch.float16, device=device), bits)

    @classmethod
    def from_tensors(cls, k_codes, v_codes, params, bits):
        """A cache around existing tensors of its format; they are adopted, not copied.  `params` may hold any scales and zero points, those of other quantizers too
        (fractions, negative numbers)."""
        if bits not in (2, 4, 8):
            raise ValueError("Only 2, 4, or 8 bits are supported.")
        if k_codes.dim() != 4 or k_codes.dtype != torch.int32 or v_codes.dtype != torch.int32 or v_codes.shape != k_codes.shape:
            raise ValueError("k_codes and v_codes must be int32 [pages, heads, page_size, head_dim * bits / 32]")
        if params.dtype != torch.float16 or tuple(params.shape) != (*k_codes.shape[:3], 4):
            raise ValueError("params must be fp16 [pages, heads, page_size, 4]")
        if min(k_codes.shape[1:]) < 1 or k_codes.shape[3] * (32 // bits) > 256:
            raise ValueError("a cache needs heads, tokens a page and a head_dim of at most 256")
        for t in (k_codes, v_codes, params):
            if not t.is_contiguous() or t.device != k_codes.device or t.data_ptr() % 16 != 0:
                raise ValueError("the cache's tensors must be contiguous, on one device and start on a 16-byte boundary")
        cache = cls.__new__(cls)
        cache._set_up(k_codes, v_codes, params, bits)
        return cache

    def _set_up(self, k_codes, v_codes, params, bits):
        self._cache = (k_codes, v_codes, params, bits)
        self.num_pages, self.num_kv_heads, self.page_size = k_codes.shape[:3]
        self.head_dim = k_codes.shape[3] * (32 // bits)
        self.device = k_codes.device
        self._shapes = (k_codes.shape, v_codes.shape, params.shape)
        self._softmax_scale = 1.0 / math.sqrt(self.head_dim)

    k_codes = property(lambda self: self._cache[0])
    v_codes = property(lambda self: self._cache[1])
    params = property(lambda self: self._cache[2])
    bits = property(lambda self: self._cache[3])

    def _tensors(self):
        tensors = self._cache[:3]
        if tuple(t.shape for t in tensors) != self._shapes or not all(t.is_contiguous() and t.device == self.device for t in tensors):
            raise RuntimeError("the cache's tensors have been changed in shape or place")
        return tuple(t.data_ptr() for t in tensors)

    def _check_slots(self, slots):
        if slots.dtype != torch.int64 or slots.dim() != 1:
            raise TypeError("slots must be an int64 vector")
        _lib.require_cuda(slots, "slots")
        if slots.device != self.device:
            raise RuntimeError(f"`slots` is on {slots.device} but the cache is on {self.device}")
        return slots if slots.is_contiguous() else slots.contiguous()

    def append(self, k, v, slots):
        """Quantises k[t], v[t] ([tokens, num_kv_heads, head_dim], fp16, bf16 or fp32; any strides of tokens and heads) into slot
        slots[t].  Slots outside the cache are skipped (padding: -1); each slot may be named once in a call.  A row with a NaN or an
        infinity, or whose scale leaves fp16's range, reads back as NaN.  Codes have no gradient: nothing is recorded."""
        if (_lib._operators or _lib.host_operators()).kv_append(*self._cache, k, v, slots):
            return
        _lib.refuse_recorders("append", traced=True)
        _lib.require_cuda(self.k_codes, "cache")
        slots = self._check_slots(slots)
        shape = (slots.shape[0], self.num_kv_heads, self.head_dim)
        for name, t in (("k", k), ("v", v)):
            _lib.require_cuda(t, name)
            if tuple(t.shape) != shape:
                raise ValueError(f"`{name}` must have shape {shape}")
            if t.dtype not in _FLOAT_DTYPES or t.dtype != k.dtype:
                raise TypeError("k and v must have one dtype: float32, float16 or bfloat16")
            if t.device != self.device:
                raise RuntimeError(f"`{name}` is on {t.device} but the cache is on {self.device}")
        if k.stride(2) != 1:
            k = k.contiguous()
        if v.stride(2) != 1:
            v = v.contiguous()
        L = _lib.lib()
        with _lib.on_device(self.device):
            rc = L.bw_kv_append(k.data_ptr(), v.data_ptr(), _lib.dtype_code(k.dtype), shape[0], k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                                slots.data_ptr(), self.num_kv_heads, self.head_dim, self.bits, self.num_pages, self.page_size, *self._tensors(),
                                _lib.raw_stream(self.device))
        _lib.check(rc)

    def append_rotated(self, q, k, v, slots, rotary, positions):
        """`append` of keys that `rotary` (a RotaryPositions) turns by `positions` on the way, and the queries q [tokens, heads, head_dim] turned alike, in
        one launch.  Returns the queries, rounded once to their dtype; q may be None.

        Keys are rotated in fp32 and quantised from there: the cache holds what `append(rotary.rotate(positions, k.float()), v.float(), slots)` would
        leave.  `positions`: int64 [tokens], or [axes, tokens].  A position outside the table gives NaN: that token's queries, and its key when it is read.  Queries
        of skipped slots are rotated too.  Nothing is recorded: a q that requires a gradient is refused where gradients are recorded, and one with a forward-mode tangent."""
        if type(rotary) is RotaryPositions:
            out = (_lib._operators or _lib.host_operators()).kv_append_rotated(*self._cache, q, k, v, slots, rotary.table, rotary._meta, positions)
            if out is not None:
                return None if q is None else out
        _lib.refuse_recorders("append_rotated", traced=True)
        _lib.require_cuda(self.k_codes, "cache")
        slots = self._check_slots(slots)
        tokens = slots.shape[0]
        shape = (tokens, self.num_kv_heads, self.head_dim)
        for name, t in (("k", k), ("v", v)):
            _lib.require_cuda(t, name)
            if tuple(t.shape) != shape:
                raise ValueError(f"`{name}` must have shape {shape}")
        for name, t in (("k", k), ("v", v), ("q", q)):
            if t is None:
                continue
            if t.dtype not in _FLOAT_DTYPES or t.dtype != k.dtype:
                raise TypeError("q, k and v must have one dtype: float32, float16 or bfloat16")
            if t.device != self.device:
                raise RuntimeError(f"`{name}` is on {t.device} but the cache is on {self.device}")
        if q is not None:
            if q.dim() != 3 or q.shape[0] != tokens or q.shape[2] != self.head_dim:
                raise ValueError(f"q must be [{tokens}, heads, {self.head_dim}]")
            _refuse_derivatives("append_rotated", q)
        if not isinstance(rotary, RotaryPositions):
            raise TypeError("rotary must be a RotaryPositions")
        if rotary.device != self.device:
            raise RuntimeError(f"`rotary` is on {rotary.device} but the cache is on {self.device}")
        if rotary.rotary_dim > self.head_dim:
            raise ValueError(f"rotary turns {rotary.rotary_dim} values but head_dim is {self.head_dim}")
        positions = rotary._positions(positions, (tokens,))
        q, k, v = (t if t is None or t.stride(2) == 1 else t.contiguous() for t in (t if t is None else t.resolve_neg() for t in (q, k, v)))
        out = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=self.device)
        L = _lib.lib()
        with _lib.on_device(self.device):
            rc = L.bw_kv_append_rotated(ctypes.byref(rotary._struct(rotary.table, positions)), *((None, 0, 0, 0, None) if q is None else (
                q.data_ptr(), q.shape[1], q.stride(0), q.stride(1), out.data_ptr())), k.data_ptr(), v.data_ptr(), _lib.dtype_code(k.dtype), tokens,
                k.stride(0), k.stride(1), v.stride(0), v.stride(1), slots.data_ptr(), self.num_kv_heads, self.head_dim, self.bits, self.num_pages, self.page_size,
                *self._tensors(), _lib.raw_stream(self.device))
        _lib.check(rc)
        return out

    def read(self, slots, dtype=torch.float16):
        """(k, v) of `slots` as [tokens, num_kv_heads, head_dim] tensors of `dtype` (fp16, bf16 or fp32): the values that the cache
        stands for, rounded once.  Slots outside the cache give zeros."""
        if dtype not in _FLOAT_DTYPES:
            raise TypeError(f"unsupported dtype {dtype}")
        both = (_lib._operators or _lib.host_operators()).kv_read(*self._cache, slots, _lib.dtype_code(dtype))
        if both is not None:
            return both
        _lib.refuse_recorders("read", traced=True)
        _lib.require_cuda(self.k_codes, "cache")
        slots = self._check_slots(slots)
        shape = (slots.shape[0], self.num_kv_heads, self.head_dim)
        k, v = torch.empty(shape, dtype=dtype, device=self.device), torch.empty(shape, dtype=dtype, device=self.device)
        L = _lib.lib()
        with _lib.on_device(self.device):
            rc = L.bw_kv_read(*self._tensors(), self.num_kv_heads, self.head_dim, self.bits, self.num_pages, self.page_size, slots.data_ptr(), shape[0],
                              k.data_ptr(), v.data_ptr(), _lib.dtype_code(dtype), _lib.raw_stream(self.device))
        _lib.check(rc)
        return k, v

    def attend(self, q, page_table, lengths, softmax_scale=None, window=None, sinks=0):
        """Attention of one new token per sequence: q [batch, heads, head_dim] (fp16 or bf16; heads a multiple of num_kv_heads, head h
        reads cache head h // (heads / num_kv_heads)) over the first lengths[b] tokens of the sequence whose pages page_table[b]
        names (int32 [batch, pages of the longest]).  Returns [batch, heads, head_dim] in q's dtype.

        `softmax_scale` defaults to head_dim ** -0.5.  The new token's own row is attended to if it has been appended and counted.  Sequences
        of length 0 (or less) give zeros.  A length that is more than the table holds, and a page outside the cache within the
        length, give NaN for that sequence; nothing is read there.  There is no gradient: a q that requires one is refused where
        gradients are recorded, and one with a forward-mode tangent.

        `window` (None: all): only the last `window` tokens of a sequence and its first `sinks` are attended to.  Pages that hold none of those are
        not looked up: they may have been given to others, and their entries of the table may be anything."""
        if softmax_scale is None:
            softmax_scale = self._softmax_scale
        if window is not None:
            return self._attend_window(q, page_table, lengths, softmax_scale, window, sinks)
        out = (_lib._operators or _lib.host_operators()).kv_attend(*self._cache, q, page_table, lengths, softmax_scale)
        if out is not None:
            return out
        q, page_table, lengths, out = self._attend_args(q, page_table, lengths)
        batch, heads = q.shape[:2]
        L = _lib.lib()
        with _lib.on_device(self.device):
            ws = _lib.workspace(self.device, L.bw_kv_attend_workspace_bytes(batch, heads, self.num_kv_heads, self.head_dim, self.page_size,
                                                                            page_table.shape[1]))
            rc = L.bw_kv_attend(q.data_ptr(), _lib.dtype_code(q.dtype), batch, heads, q.stride(0), q.stride(1), *self._tensors(), self.bits, self.num_pages,
                                self.page_size, self.num_kv_heads, self.head_dim, page_table.data_ptr(), page_table.stride(0), page_table.shape[1],
                                lengths.data_ptr(), float(softmax_scale), out.data_ptr(), None if ws is None else ws.data_ptr(),
                                0 if ws is None else ws.numel(), _lib.raw_stream(self.device))
        _lib.check(rc)
        return out

    def _attend_window(self, q, page_table, lengths, softmax_scale, window, sinks):
        try:
            window, sinks = min(operator.index(window), 2 ** 31), min(operator.index(sinks), 2 ** 31)
        except TypeError:
            window = -1
        if window < 0 or sinks < 0:
            raise ValueError("window and sinks must be numbers of tokens, 0 or more")
        out = (_lib._operators or _lib.host_operators()).kv_attend(*self._cache, q, page_table, lengths, softmax_scale, window, sinks)
        if out is not None:
            return out
        q, page_table, lengths, out = self._attend_args(q, page_table, lengths)
        batch, heads = q.shape[:2]
        L = _lib.lib()
        with _lib.on_device(self.device):
            ws = _lib.workspace(self.device, L.bw_kv_attend_window_workspace_bytes(batch, heads, self.num_kv_heads, self.head_dim, self.page_size,
                                                                                   page_table.shape[1], window, sinks))
            rc = L.bw_kv_attend_window(q.data_ptr(), _lib.dtype_code(q.dtype), batch, heads, q.stride(0), q.stride(1), *self._tensors(), self.bits, self.num_pages,
                                       self.page_size, self.num_kv_heads, self.head_dim, page_table.data_ptr(), page_table.stride(0), page_table.shape[1],
                                       lengths.data_ptr(), window, sinks, float(softmax_scale), out.data_ptr(), None if ws is None else ws.data_ptr(),
                                       0 if ws is None else ws.numel(), _lib.raw_stream(self.device))
        _lib.check(rc)
        return out

    def _attend_args(self, q, page_table, lengths):
        """Checked arguments of a call of attention as the kernels take them, and its output."""
        _lib.refuse_recorders("attend", traced=True)
        _lib.require_cuda(q, "q")
        if q.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"attend: unsupported dtype {q.dtype} (float16/bfloat16)")
        _refuse_derivatives("attend", q)
        if q.dim() != 3 or q.shape[2] != self.head_dim or q.shape[1] < 1 or q.shape[1] % self.num_kv_heads != 0:
            raise ValueError(f"q must be [batch, heads, {self.head_dim}] with a multiple of {self.num_kv_heads} heads")
        if page_table.dtype != torch.int32 or lengths.dtype != torch.int32:
            raise TypeError("page_table and lengths must be int32")
        batch, heads = q.shape[:2]
        if page_table.dim() != 2 or page_table.shape[0] != batch or tuple(lengths.shape) != (batch,):
            raise ValueError(f"page_table must be [{batch}, pages] and lengths [{batch}]")
        for name, t in (("q", q), ("page_table", page_table), ("lengths", lengths)):
            if t.device != self.device:
                raise RuntimeError(f"`{name}` is on {t.device} but the cache is on {self.device}")
        if q.stride(2) != 1:
            q = q.contiguous()
        if page_table.stride(1) != 1:
            page_table = page_table.contiguous()
        if not lengths.is_contiguous():
            lengths = lengths.contiguous()
        return q, page_table, lengths, torch.empty((batch, heads, self.head_dim), dtype=q.dtype, device=self.device)

    def __repr__(self):
        return (f"QuantizedKVCache(num_pages={self.num_pages}, page_size={self.page_size}, num_kv_heads={self.num_kv_heads}, "
                f"head_dim={self.head_dim}, bits={self.bits})")
