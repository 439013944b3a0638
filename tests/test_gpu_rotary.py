"""Rotary positions, by themselves with gradients and on the way into the quantised cache: against fp32 steps bit for bit, and 64-bit sums."""
import math

import pytest
import torch

from bitween_b200 import QuantizedKVCache, RotaryPositions
from bitween_b200.kernels import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rows(shape, seed, dtype):
    g = _gen(seed)
    x = torch.randn(shape, generator=g, device=DEV) * (0.5 + torch.rand(shape[-1], generator=g, device=DEV))
    return (x + 0.3 * torch.randn(shape[-1], generator=g, device=DEV)).to(dtype)


def turned(r, positions, x, back=False):
    """The definition's fp32 steps: products and sums rounded once each, by torch's elementwise kernels."""
    pairs, x = r.rotary_dim // 2, x.float()
    axis = torch.tensor(r.axes, device=DEV)
    at = positions[None].expand(r.num_axes, *positions.shape) if positions.dim() == x.dim() - 2 else positions
    at = at[axis].movedim(0, -1)                                       # [..., pairs]
    ok = (at >= 0) & (at < r.max_positions)
    t = r.table[at.clamp(0, r.max_positions - 1), torch.arange(pairs, device=DEV)].masked_fill(~ok[..., None], math.nan)
    c, s = t[..., None, :, 0], t[..., None, :, 1]
    s = -s if back else s
    y = x.clone()
    a, b = (x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]) if r.interleaved else (x[..., :pairs], x[..., pairs:2 * pairs])
    first, second = a * c - b * s, b * c + a * s
    if r.interleaved:
        y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = first, second
    else:
        y[..., :pairs], y[..., pairs:2 * pairs] = first, second
    return y


def same(a, b):
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


# dim, rotary dim, axes of the pairs, interleaved
FORMS = [(128, 128, None, False), (128, 128, (16, 24, 24), False), (128, 128, "mixed", False), (64, 64, None, True), (64, 32, None, False), (256, 256, (32, 96), False),
         (256, 64, (8, 16, 8), True), (128, 64, "mixed", True), (80, 80, None, False), (96, 32, None, False), (128, 20, None, True), (192, 192, None, False),
         (64, 16, None, False), (50, 2, None, False), (112, 112, (10, 46), False), (7, 6, None, True), (512, 256, None, False)]


def _rotary(rotary, axes, interleaved, most=700):
    if axes == "mixed":                                                # three axes in turn
        return RotaryPositions(rotary, most, axes=[j % 3 for j in range(rotary // 2)], interleaved=interleaved)
    return RotaryPositions(rotary, most, sections=axes, interleaved=interleaved)


@pytest.mark.parametrize("dim,rotary,axes,interleaved", FORMS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_rotate(dim, rotary, axes, interleaved, dtype):
    r = _rotary(rotary, axes, interleaved)
    for tokens, heads, kv_heads in ((1, 1, 1), (3, 32, 8), (37, 5, 2), (129, 12, 12)):
        p = torch.randint(0, 700, (r.num_axes, tokens), generator=_gen(1), device=DEV)
        if r.num_axes == 1:
            p = p[0]
        q, k = _rows((tokens, heads, dim), 2, dtype), _rows((tokens, kv_heads, dim), 3, dtype)
        yq, yk = r.rotate(p, q, k)
        assert same(yq, turned(r, p, q).to(dtype)) and same(yk, turned(r, p, k).to(dtype))
        assert same(r.rotate(p, k), yk)
        # against 64 bits: two products and their sum, 2^-24 of each, and the result's rounding
        angle = (p[None] if p.dim() == 1 else p)[torch.tensor(r.axes, device=DEV)].T.double() * 10000.0 ** (-torch.arange(rotary // 2, device=DEV, dtype=torch.float64) * 2 / rotary)
        z = torch.complex(*((q[..., 0:rotary:2].double(), q[..., 1:rotary:2].double()) if interleaved else (q[..., :rotary // 2].double(), q[..., rotary // 2:rotary].double())))
        want = z * torch.polar(torch.ones_like(angle), angle)[:, None]
        got = torch.complex(*((yq[..., 0:rotary:2].double(), yq[..., 1:rotary:2].double()) if interleaved else (yq[..., :rotary // 2].double(), yq[..., rotary // 2:rotary].double())))
        for part in ("real", "imag"):
            w = getattr(want, part)
            # cosine and sine: 2^-25 of 1 each, products 2^-24: together at most 2^-23 of |a| + |b| <= sqrt(2) |z|; then the rounding (of fp16 also its smallest steps)
            slack = 2.0 ** -22 * want.abs()
            assert bool(((getattr(got, part) - w).abs() <= slack + torch.finfo(dtype).eps / 2 * (w.abs() + slack) + 2.0 ** -25).all())


@pytest.mark.parametrize("dim,rotary,axes,interleaved", FORMS[:8] + [(80, 80, None, False)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_gradients_are_turned_back(dim, rotary, axes, interleaved, dtype):
    r = _rotary(rotary, axes, interleaved)
    p = torch.randint(0, 700, (r.num_axes, 45), generator=_gen(4), device=DEV)
    p = p[0] if r.num_axes == 1 else p
    q, k = _rows((45, 6, dim), 5, dtype).requires_grad_(), _rows((45, 2, dim), 6, dtype).requires_grad_()
    yq, yk = r.rotate(p, q, k)
    with torch.no_grad():
        assert same(yq.detach(), r.rotate(p, q)) and same(yk.detach(), r.rotate(p, k))
    gq, gk = _rows(yq.shape, 7, dtype), _rows(yk.shape, 8, dtype)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk), retain_graph=True)
    assert same(dq, turned(r, p, gq, back=True).to(dtype)) and same(dk, turned(r, p, gk, back=True).to(dtype))
    (only,) = torch.autograd.grad(yk, k, gk, retain_graph=True)           # one output that is not used, an expanded gradient
    assert same(only, dk)
    (broad,) = torch.autograd.grad(yq, q, torch.ones((), dtype=dtype, device=DEV).expand(yq.shape))
    assert same(broad, turned(r, p, torch.ones_like(gq), back=True).to(dtype))
    if dtype == torch.float32:
        # linear: a difference of values is the gradient's product but for roundings of 2^-24 of 100 values of some units
        d = _rows(q.shape, 9, dtype)
        with torch.no_grad():
            diff = ((r.rotate(p, q + d).double() - r.rotate(p, q).double()) * gq.double()).sum()
        assert abs(float(diff - (dq.double() * d.double()).sum())) <= 2.0 ** -22 * float((gq.double().abs() * (q.detach().double().abs() + d.double().abs() + 1)).sum())


def test_strides_shapes_and_positions():
    r = _rotary(128, (16, 24, 24), False)
    fused = _rows((2, 33, 20 * 128 + 8), 10, torch.bfloat16)
    q = fused[..., :16 * 128].unflatten(-1, (16, 128))
    k = fused[..., 16 * 128:20 * 128].unflatten(-1, (4, 128))
    p = torch.randint(0, 700, (3, 2, 33), generator=_gen(11), device=DEV)
    yq, yk = r.rotate(p, q, k)
    assert same(yq, turned(r, p, q).to(q.dtype)) and same(yk, turned(r, p, k).to(q.dtype)) and yq.is_contiguous()
    assert same(r.rotate(p[1], q), turned(r, p[1], q).to(q.dtype))                 # one position for all axes
    assert same(r.rotate(p.permute(1, 2, 0).contiguous().permute(2, 0, 1), q), yq)
    assert same(r.rotate(p[:1].expand(3, 2, 33), q), turned(r, p[0], q).to(q.dtype))
    heads_last = q.transpose(2, 3).contiguous().transpose(2, 3)
    assert same(r.rotate(p, heads_last), yq)
    odd = fused.flatten()[1:1 + 33 * 4 * 128].view(33, 4, 128)                     # rows off a 16-byte boundary
    assert same(r.rotate(p[:, 0], odd), turned(r, p[:, 0], odd).to(odd.dtype))
    one = r.rotate(p[:, 0, 0], odd[0])                                             # no leading dimension
    assert same(one, turned(r, p[:, 0, :1], odd[:1])[0].to(odd.dtype))
    assert r.rotate(p[:, :0], q[:0]).shape == (0, 33, 16, 128)
    far = p.clone()
    far[0, 0, 5], far[1, 1, 7], far[2, 1, 8] = 700, -1, 2 ** 40
    got, want = r.rotate(far, q), turned(r, far, q).to(q.dtype)
    assert same(got, want) and int(got.isnan().any(-1).any(-1).sum()) == 3
    assert bool(got[0, 5, :, 16:64].isfinite().all()) and bool(got[0, 5, :, :16].isnan().all())
    assert _lib.lib().bw_device_status() == 0


def test_many_rows():
    """More tokens than one wave of CTAs, rows of 40 heads."""
    r = _rotary(128, None, False)
    p = torch.randint(0, 700, (9001,), generator=_gen(12), device=DEV)
    q, k = _rows((9001, 32, 128), 13, torch.float16), _rows((9001, 8, 128), 14, torch.float16)
    for x, y in zip((q, k), r.rotate(p, q, k)):
        assert same(y, turned(r, p, x).half())


def test_infinities_stay_in_their_pair():
    r = _rotary(64, None, False)
    p = torch.arange(9, device=DEV)
    x = _rows((9, 2, 64), 15, torch.float16)
    x[3, 1, 5], x[4, 0, 40] = math.inf, math.nan
    y = r.rotate(p, x)
    assert same(y, turned(r, p, x).half())
    bad = ~y.isfinite()
    assert bool(bad[3, 1, [5, 37]].all()) and bool(bad[4, 0, [8, 40]].all()) and int(bad.sum()) == 4


def _cache(pages, page, heads, dim, bits):
    cache = QuantizedKVCache(pages, page, heads, dim, bits=bits, device=DEV)
    cache.k_codes.fill_(-1)
    cache.v_codes.fill_(-1)
    cache.params.fill_(7)
    return cache


@pytest.mark.parametrize("dim,rotary,axes,interleaved", FORMS[:9] + [(96, 32, None, False), (192, 192, None, False), (16, 16, None, False), (48, 16, None, True)])
@pytest.mark.parametrize("bits", [2, 4, 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_append_rotated(dim, rotary, axes, interleaved, bits, dtype):
    r = _rotary(rotary, axes, interleaved)
    for tokens, heads, kv_heads, page in ((1, 4, 2, 16), (61, 6, 3, 16), (200, 8, 1, 7)):
        fused = _rows((tokens, heads + 2 * kv_heads, dim), 20, dtype)
        q, k, v = fused[:, :heads], fused[:, heads:heads + kv_heads], fused[:, heads + kv_heads:]
        k[tokens // 2] = 0
        p = torch.randint(0, 700, (r.num_axes, tokens), generator=_gen(21), device=DEV)
        p = p[0] if r.num_axes == 1 else p
        pages = -(-tokens // page) + 3
        slots = torch.randperm(pages * page, generator=_gen(22), device=DEV)[:tokens]
        if tokens > 20:
            slots[3], slots[9] = -1, pages * page                                  # padding: skipped, their queries rotated all the same
        cache, plain = _cache(pages, page, kv_heads, dim, bits), _cache(pages, page, kv_heads, dim, bits)
        out = cache.append_rotated(q, k, v, slots, r, p)
        plain.append(turned(r, p, k), v.float(), slots)
        assert same(out, turned(r, p, q).to(dtype)) and out.is_contiguous()
        for name in ("k_codes", "v_codes", "params"):
            assert torch.equal(getattr(cache, name), getattr(plain, name)), name
        assert cache.append_rotated(None, k, v, slots, r, p) is None
        assert torch.equal(cache.k_codes, plain.k_codes) and torch.equal(cache.params, plain.params)
    assert _lib.lib().bw_device_status() == 0


def test_append_rotated_of_strided_and_odd_tensors_and_bad_positions():
    r = _rotary(128, (16, 24, 24), False)
    cache, plain = _cache(9, 16, 2, 128, 4), _cache(9, 16, 2, 128, 4)
    big = _rows((140 * 12 * 128 + 1,), 23, torch.float16)
    q, k, v = big[1:].view(140, 12, 128)[:, :6], big[1:].view(140, 12, 128)[:, 6:8], big[1:].view(140, 12, 128)[:, 8:10]
    p = torch.randint(0, 700, (3, 140), generator=_gen(24), device=DEV)
    p[1, 7], p[0, 9] = 700, -5
    slots = torch.arange(140, device=DEV)
    out = cache.append_rotated(q, k, v, slots, r, p)
    plain.append(turned(r, p, k), v.float(), slots)
    assert same(out, turned(r, p, q).half())
    rk, rv = cache.read(slots)
    wk, wv = plain.read(slots)
    assert same(rk, wk) and same(rv, wv) and bool(rk[[7, 9]].isnan().all()) and bool(rv.isfinite().all())
    heads_last = k.transpose(1, 2).contiguous().transpose(1, 2)
    again = _cache(9, 16, 2, 128, 4)
    assert same(again.append_rotated(q.contiguous(), heads_last, v.contiguous(), slots, r, p), out) and torch.equal(again.k_codes, cache.k_codes)
    assert cache.append_rotated(q[:0], k[:0], v[:0], slots[:0], r, p[:, :0]).shape == (0, 6, 128)
    # rows with an infinity, and of more than fp16's range, read back as NaN
    k = k.float().clone()
    k[0, 0, 3], k[1, 1, 70], k[2] = math.inf, 1e9, k[2] * 1e-9
    cache.append_rotated(None, k, v.float(), slots, r, p)
    plain.append(turned(r, p, k), v.float(), slots)
    assert same(cache.read(slots)[0], plain.read(slots)[0]) and torch.equal(cache.k_codes, plain.k_codes)
    assert bool(cache.read(slots[:2])[0][[0, 1], [0, 1]].isnan().all())


def test_offsets_past_32_bits():
    """Queries whose rows lie more than 2^31 values behind the first one."""
    r = _rotary(64, None, False)
    x = torch.empty((70000, 480, 64), dtype=torch.float16, device=DEV)
    x[::35000] = _rows((2, 480, 64), 25, torch.float16)
    x[-1] = _rows((480, 64), 26, torch.float16)
    p = torch.arange(70000, device=DEV) % 700
    y = r.rotate(p, x)
    at = torch.tensor([0, 35000, 69999], device=DEV)
    assert same(y[at], turned(r, p[at], x[at]).half())
    del y
    cache, plain = _cache(1, 16, 480, 64, 8), _cache(1, 16, 480, 64, 8)
    rows = x[34999::35000]                                                          # (2 tokens, 35000 rows apart)
    rows.copy_(_rows(rows.shape, 27, torch.float16))
    slots = torch.tensor([3, 5], device=DEV)
    out = cache.append_rotated(rows, rows, rows, slots, r, p[:2])
    plain.append(turned(r, p[:2], rows), rows.float(), slots)
    assert same(out, turned(r, p[:2], rows).half()) and torch.equal(cache.k_codes, plain.k_codes) and torch.equal(cache.v_codes, plain.v_codes)
