"""The checks of the arguments of rotary positions, rotated appends, windowed attention and log probabilities, which need no GPU."""
import ctypes

import pytest
import torch

from bitween_b200 import QuantizedKVCache, RotaryPositions, token_log_probs
from bitween_b200.kernels import _lib

P = 1 << 20      # an aligned address that no call here reaches


def _rotary(table=P, most=100, dim=64, num_axes=1, axes=None, positions=P):
    return ctypes.byref(_lib.Rotary(table, most, dim, 0, num_axes, axes, positions, 0))


def test_rotate_checks_its_arguments():
    L = _lib.lib()

    def rotate(r=None, tokens=4, dim=64, dtype=1, x=P, heads=2, out=P, y=P, heads1=1):
        return L.bw_rotate(_rotary() if r is None else r, tokens, dim, dtype, 0, x, heads, 128, 64, out, y, heads1, 128, 64, P, None)

    assert L.bw_rotate(None, 4, 64, 1, 0, P, 2, 128, 64, P, None, 0, 0, 0, None, None) == 6
    for bad in (_rotary(dim=63), _rotary(dim=0), _rotary(dim=258), _rotary(dim=128), _rotary(num_axes=0), _rotary(num_axes=256), _rotary(most=-1),
                _rotary(num_axes=2, axes=bytes([0, 1] * 15 + [2, 0]))):
        assert rotate(r=bad) == 3
    assert rotate(tokens=-1) == 3 and rotate(tokens=1 << 40) == 3 and rotate(heads=-1) == 3 and rotate(heads=1 << 21) == 3
    assert rotate(dtype=3) == 4 and rotate(dtype=9) == 4
    assert rotate(r=_rotary(table=P + 8)) == 5 and rotate(r=_rotary(positions=P + 4)) == 5 and rotate(x=P + 1) == 5 and rotate(out=P + 1) == 5
    assert rotate(r=_rotary(table=None)) == 6 and rotate(r=_rotary(positions=None)) == 6 and rotate(x=None) == 6 and rotate(out=None) == 6 and rotate(y=None) == 6
    assert rotate(tokens=0) == 0 and rotate(heads=0, heads1=0) == 0 and rotate(tokens=0, r=_rotary(positions=None)) == 0


def test_append_rotated_checks_its_arguments():
    L = _lib.lib()

    def append(r=None, q=P, q_heads=4, q_out=P, k=P, dtype=1, tokens=4, heads=2, dim=64, bits=4, slots=P, codes=P, pages=3):
        return L.bw_kv_append_rotated(_rotary() if r is None else r, q, q_heads, 256, 64, q_out, k, P, dtype, tokens, 128, 64, 128, 64, slots, heads, dim, bits, pages, 16,
                                      codes, P, P, None)

    assert append(bits=3) == 1
    assert append(dim=60) == 3 and append(heads=0) == 3 and append(tokens=-1) == 3 and append(tokens=1 << 40) == 3 and append(q_heads=-1) == 3
    assert append(r=_rotary(dim=128)) == 3 and append(r=_rotary(dim=30, num_axes=1, axes=bytes([1] * 15))) == 3
    assert append(dtype=3) == 4
    assert append(k=P + 1) == 5 and append(q=P + 1) == 5 and append(q_out=P + 1) == 5 and append(codes=P + 4) == 5 and append(slots=P + 4) == 5
    assert append(k=None) == 6 and append(q=None) == 6 and append(q_out=None) == 6 and append(slots=None) == 6 and append(codes=None) == 6
    assert append(tokens=0) == 0


def test_windowed_attention_checks_its_arguments():
    L = _lib.lib()

    def attend(dtype=1, batch=2, heads=4, kv_heads=2, dim=64, table=P, wide=4, q=P, lengths=P, ws=P, size=1 << 40, window=100, sinks=4):
        return L.bw_kv_attend_window(q, dtype, batch, heads, heads * dim, dim, P, P, P, 4, 3, 16, kv_heads, dim, table, 4, wide, lengths, window, sinks, 0.1, P, ws, size,
                                     None)

    assert attend(window=-1) == 3 and attend(sinks=-1) == 3 and attend(heads=3) == 3 and attend(wide=1 << 31) == 3
    assert attend(dtype=0) == 4 and attend(q=None) == 6 and attend(table=None) == 6 and attend(lengths=None) == 6
    assert attend(q=P + 1) == 5 and attend(table=P + 2) == 5
    assert attend(batch=0) == 0
    need = L.bw_kv_attend_window_workspace_bytes(64, 4, 2, 64, 16, 1 << 20, 1 << 20, 4)
    assert need > 0
    assert attend(batch=64, wide=1 << 20, window=1 << 20, ws=None) == 7 and attend(batch=64, wide=1 << 20, window=1 << 20, size=need - 1) == 7
    assert attend(batch=64, wide=1 << 20, window=1 << 20, ws=P + 8) == 5
    assert L.bw_kv_attend_window_workspace_bytes(2, 4, 2, 64, 16, 4, -1, 4) == 0 and L.bw_kv_attend_window_workspace_bytes(0, 4, 2, 64, 16, 4, 1, 4) == 0


def test_log_probs_check_their_arguments():
    L = _lib.lib()

    def forward(x=P, dtype=1, rows=4, vocab=100, tokens=P, lp=P, h=P, top=5, top_lp=P, top_t=P, stats=P):
        return L.bw_token_log_probs(x, dtype, rows, vocab, vocab, tokens, lp, h, top, top_lp, top_t, stats, None)

    assert forward(dtype=3) == 4
    assert forward(rows=-1) == 3 and forward(rows=1 << 40) == 3 and forward(vocab=0) == 3 and forward(vocab=1 << 29) == 3 and forward(top=33) == 3 and forward(top=-1) == 3
    assert forward(vocab=4) == 3
    assert forward(x=None) == 6 and forward(tokens=None) == 6 and forward(lp=None) == 6 and forward(top_lp=None) == 6 and forward(top_t=None) == 6
    assert forward(x=P + 1) == 5 and forward(tokens=P + 4) == 5 and forward(lp=P + 2) == 5 and forward(h=P + 2) == 5 and forward(stats=P + 8) == 5 and forward(top_t=P + 4) == 5
    assert forward(rows=0) == 0

    def backward(x=P, dtype=1, rows=4, vocab=100, tokens=P, stats=P, g=P, e=P, top=5, top_t=P, g_top=P, grad=P):
        return L.bw_token_log_probs_grad(x, dtype, rows, vocab, vocab, tokens, stats, g, e, top, top_t, g_top, grad, None)

    assert backward(dtype=9) == 4 and backward(rows=-1) == 3 and backward(top=40) == 3
    assert backward(x=None) == 6 and backward(stats=None) == 6 and backward(grad=None) == 6 and backward(tokens=None) == 6 and backward(top_t=None) == 6
    assert backward(x=P + 1) == 5 and backward(stats=P + 8) == 5 and backward(grad=P + 1) == 5 and backward(g=P + 2) == 5
    assert backward(rows=0) == 0


def test_refusals():
    for args in ((0, 4), (7, 4), (258, 4), (64, 0)):
        with pytest.raises(ValueError):
            RotaryPositions(*args, device="cpu")
    for kw in ({"sections": (8, 8)}, {"sections": (40, -8)}, {"axes": [0] * 31}, {"axes": [-1] * 32}, {"sections": (32,), "axes": [0] * 32}, {"inv_freq": [1.0] * 8}, {"axes": [255] * 32},
               {"sections": ()}):
        with pytest.raises(ValueError):
            RotaryPositions(64, 4, device="cpu", **kw)
    r = RotaryPositions(64, 50, sections=(8, 12, 12), device="cpu")
    assert r.table.shape == (50, 32, 2) and r.num_axes == 3 and r.axes == (0,) * 8 + (1,) * 12 + (2,) * 12 and "num_axes=3" in repr(r)
    angle = torch.arange(50, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    # (cosines are at most 1: rounded to fp32 they are off by 2^-25, and 64-bit angles of up to 50 by 2^-48)
    assert bool(((r.table[..., 0].double() - angle.cos()).abs() <= 2.0 ** -25 + 2.0 ** -46).all())
    assert torch.equal(RotaryPositions(64, 50, factor=2.0, device="cpu").table, 2 * RotaryPositions(64, 50, device="cpu").table)
    x, p = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError):
        r.rotate(p, x)                                  # no CPU path
    with pytest.raises(ValueError):
        r.rotate(p)
    cache = QuantizedKVCache(4, 16, 2, 64, bits=4, device="cpu")
    with pytest.raises(RuntimeError):
        cache.append_rotated(x, x, x, p, r, p)
    table, lengths = torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    for kw in ({"window": -1}, {"window": 4, "sinks": -1}, {"window": 1.5}, {"window": 4, "sinks": None}):
        with pytest.raises(ValueError):
            cache.attend(x.half(), table, lengths, **kw)
    with pytest.raises(RuntimeError):
        cache.attend(x.half(), table, lengths, window=4)
    with pytest.raises(RuntimeError):
        token_log_probs(torch.zeros(3, 50), p)


@pytest.mark.gpu
def test_refusals_of_tensors_on_the_gpu():
    dev = "cuda"
    r = RotaryPositions(64, 50, sections=(8, 12, 12))
    x, p = torch.zeros(3, 2, 64, device=dev).half(), torch.zeros(3, dtype=torch.int64, device=dev)
    cache = QuantizedKVCache(4, 16, 2, 64, bits=4, device=dev)
    logits = torch.zeros(3, 50, device=dev)
    wider = RotaryPositions(128, 50)
    changed = RotaryPositions(64, 50)
    changed.table = changed.table[:20]
    for error, call in (
            (TypeError, lambda: r.rotate(p.int(), x)), (ValueError, lambda: r.rotate(p[:2], x)), (ValueError, lambda: r.rotate(p.expand(2, 3), x)),
            (RuntimeError, lambda: r.rotate(p.cpu(), x)), (TypeError, lambda: r.rotate(p, x.double())), (TypeError, lambda: r.rotate(p, x, x.float())),
            (ValueError, lambda: r.rotate(p, x, x[:2])), (ValueError, lambda: r.rotate(p, x[..., :32])), (ValueError, lambda: r.rotate(p, x, x, x)),
            (RuntimeError, lambda: r.rotate(p, x.cpu())), (ValueError, lambda: wider.rotate(p, x)), (RuntimeError, lambda: changed.rotate(p, x)),
            (TypeError, lambda: cache.append_rotated(x, x, x, p.int(), r, p)), (ValueError, lambda: cache.append_rotated(x[:2], x, x, p, r, p)),
            (TypeError, lambda: cache.append_rotated(x.float(), x, x, p, r, p)), (ValueError, lambda: cache.append_rotated(x, x, x[:, :1], p, r, p)),
            (TypeError, lambda: cache.append_rotated(x, x, x, p, None, p)), (ValueError, lambda: cache.append_rotated(x, x, x, p, wider, p)),
            (TypeError, lambda: cache.append_rotated(x, x, x, p, r, p.int())), (ValueError, lambda: cache.append_rotated(x, x, x, p, r, p[:1])),
            (RuntimeError, lambda: cache.append_rotated(x, x, x, p, changed, p)),
            (ValueError, lambda: cache.append_rotated(x.clone().requires_grad_(), x, x, p, r, p)),
            (TypeError, lambda: token_log_probs(logits.double(), p)), (TypeError, lambda: token_log_probs(logits, p.int())), (ValueError, lambda: token_log_probs(logits, p[:2])),
            (RuntimeError, lambda: token_log_probs(logits, p.cpu())), (ValueError, lambda: token_log_probs(logits, p, top=33)), (ValueError, lambda: token_log_probs(logits, p, top=-1)),
            (ValueError, lambda: token_log_probs(logits[:, :4], p, top=5)), (ValueError, lambda: token_log_probs(logits[:, :0], p))):
        with pytest.raises(error):
            call()
