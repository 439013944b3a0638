"""Attention over the quantised cache with a sliding window and sinks, against 64-bit sums over the visible tokens."""
import math

import pytest
import torch

from bitween_b200 import QuantizedKVCache
from bitween_b200.kernels import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rows(shape, seed):
    g = _gen(seed)
    x = torch.randn(shape, generator=g, device=DEV) * (0.5 + torch.rand(shape[-1], generator=g, device=DEV))
    return (x + 0.3 * torch.randn(shape[-1], generator=g, device=DEV)).half()


def _visible(n, window, sinks):
    t = torch.arange(max(n, 0), device=DEV)
    return t[(t < sinks) | (t >= n - window)]


def _filled(lengths, heads, dim, bits, page, window, sinks, seed):
    """A cache that holds the visible tokens alone: pages without one are named by numbers outside the cache, and every other row reads as NaN."""
    wide = max(1, -(-max(lengths) // page))
    seen = [_visible(n, window, sinks) for n in lengths]
    held = torch.zeros(len(lengths), wide, dtype=torch.bool, device=DEV)
    for b, t in enumerate(seen):
        held[b, t // page] = True
    pages = int(held.sum()) + 2
    cache = QuantizedKVCache(pages, page, heads, dim, bits=bits, device=DEV)
    cache.params.fill_(math.nan)
    table = torch.full(held.shape, -1, dtype=torch.int64, device=DEV)
    table[:, ::3] = pages + 5
    table[held] = torch.randperm(pages, generator=_gen(seed), device=DEV)[:pages - 2]
    slots = [table[b, t // page] * page + t % page for b, t in enumerate(seen)]
    for part in torch.cat(slots).split(1 << 16):
        shape = (part.numel(), heads, dim)
        cache.append(_rows(shape, seed + 1), _rows(shape, seed + 2), part)
    return cache, table.to(torch.int32), torch.tensor(lengths, dtype=torch.int32, device=DEV), slots


def _attended(cache, q, slots, alpha):
    """(outputs, sums of w |v|) in 64 bits over the rows `slots` of each sequence."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(out)
    group = q.shape[1] // cache.num_kv_heads
    for b, s in enumerate(slots):
        if not s.numel():
            continue
        k, v = (x.double().repeat_interleave(group, 1) for x in cache.read(s, dtype=torch.float32))
        w = torch.softmax(torch.einsum("hd,thd->ht", q[b].double(), k) * alpha, -1)
        out[b] = torch.einsum("ht,thd->hd", w, v)
        size[b] = torch.einsum("ht,thd->hd", w, v.abs())
    return out, size


def _check(got, want, size):
    """The result's own rounding; scores of some units have fp32 errors of less than 2^-17 (256 products, 2^-24 of a sum of up to 30 each, in blocks of 16), and the weights with them."""
    half = torch.finfo(got.dtype).eps / 2
    slack = 2.0 ** -14 * size
    assert bool(((got.double() - want).abs() <= half * (want.abs() + slack) + slack + 2.0 ** -25).all())


LAYOUTS = [(12, 12, 64, 8, 16), (8, 2, 128, 4, 16), (10, 2, 128, 2, 48), (16, 2, 128, 8, 64), (32, 2, 256, 4, 32), (24, 2, 64, 2, 16), (34, 1, 128, 4, 16), (4, 4, 128, 4, 32),
           (6, 3, 80, 4, 16), (4, 2, 128, 8, 7), (4, 1, 256, 2, 16)]


@pytest.mark.parametrize("heads,kv_heads,dim,bits,page", LAYOUTS)
@pytest.mark.parametrize("window,sinks", [(64, 4), (1, 0), (0, 5), (17, 16), (200, 33), (333, 1), (5000, 3), (16, 0), (31, 48), (0, 0)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_short_and_long_sequences(heads, kv_heads, dim, bits, page, window, sinks, dtype):
    lengths = [700, 0, 1, 5, 16, 17, 203, 64, 65, 340, 1000]
    cache, table, n, slots = _filled(lengths, kv_heads, dim, bits, page, window, sinks, 3)
    q = torch.randn(len(lengths), heads, dim, generator=_gen(4), device=DEV).to(dtype)
    got = cache.attend(q, table, n, window=window, sinks=sinks)
    assert got.dtype == dtype and got.shape == q.shape
    want, size = _attended(cache, q, slots, dim ** -0.5)
    _check(got, want, size)
    if window + sinks == 0:
        assert not bool(got.any())
    assert torch.equal(got, cache.attend(q, table, n, window=window, sinks=sinks))          # no sum depends on the order of arrival
    assert _lib.lib().bw_device_status() == 0


@pytest.mark.parametrize("lengths,window,sinks,heads,kv_heads,dim,bits,page", [
    ([8192, 3000, 1, 999, 1005, 0, 4100, 7777] * 3, 1000, 4, 32, 8, 128, 4, 16),
    ([131071], 4096, 64, 8, 2, 128, 8, 64),                     # one long document: its window is shared by many CTAs
    ([131072, 60000], 8192, 100, 4, 4, 64, 2, 32),
    ([30011, 4, 16000], 5000, 3000, 16, 1, 256, 4, 16),         # sinks as many as the window
    ([2000] * 40, 777, 0, 10, 2, 128, 8, 16),
    ([50000, 100], 1, 20001, 12, 6, 64, 4, 48),
])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_windows_of_long_sequences(lengths, window, sinks, heads, kv_heads, dim, bits, page, dtype):
    cache, table, n, slots = _filled(lengths, kv_heads, dim, bits, page, window, sinks, 5)
    q = torch.randn(len(lengths), heads, dim, generator=_gen(6), device=DEV).to(dtype)
    got = cache.attend(q, table, n, window=window, sinks=sinks)
    _check(got, *_attended(cache, q, slots, dim ** -0.5))
    assert torch.equal(got, cache.attend(q, table, n, window=window, sinks=sinks))
    assert _lib.lib().bw_device_status() == 0


@pytest.mark.parametrize("heads,kv_heads,dim,bits,page", LAYOUTS)
def test_a_window_that_holds_everything_is_attention_without_one(heads, kv_heads, dim, bits, page):
    lengths = [300, 0, 17, 123]
    cache, table, n, slots = _filled(lengths, kv_heads, dim, bits, page, 10 ** 6, 0, 7)
    q = torch.randn(4, heads, dim, generator=_gen(8), device=DEV).half()
    plain = cache.attend(q, table, n)
    want, size = _attended(cache, q, slots, dim ** -0.5)
    for window, sinks in ((300, 0), (2 ** 40, 7), (0, 300), (150, 150), (2 ** 31 - 1, 2 ** 31 - 1)):
        got = cache.attend(q, table, n, window=window, sinks=sinks)
        _check(got, want, size)
    assert torch.equal(cache.attend(q, table, n, sinks=5), plain)                            # (no window: all is visible)


@pytest.mark.parametrize("dim,page", [(128, 16), (64, 64), (80, 16)])
def test_bad_pages_and_lengths(dim, page):
    lengths = [400, 400, 400, 400, 400, 400]
    window, sinks = 70, 20
    cache, table, n, slots = _filled(lengths, 2, dim, 4, page, window, sinks, 9)
    q = torch.randn(6, 4, dim, generator=_gen(10), device=DEV).half()
    want, size = _attended(cache, q, slots, dim ** -0.5)
    table[1, 399 // page] = cache.num_pages                            # in the window
    table[2, 0] = -1                                                   # in the sinks
    n[3] = table.shape[1] * page + 1                                   # more than the table holds
    n[4] = -7
    got = cache.attend(q, table, n, window=window, sinks=sinks)
    assert bool(got[[1, 2, 3]].isnan().all()) and bool((got[4] == 0).all())
    _check(got[[0, 5]], want[[0, 5]], size[[0, 5]])
    n.fill_(2 ** 31 - 1)                                               # (and far more)
    assert bool(cache.attend(q, table, n, window=window, sinks=sinks).isnan().all())
    assert bool(cache.attend(q, table, n, window=0, sinks=0).isnan().all())
    assert bool(cache.attend(q, table[:, :0], n, window=window, sinks=sinks).isnan().all())
    assert not bool(cache.attend(q, table[:, :0], torch.zeros_like(n), window=window, sinks=sinks).any())
    assert cache.attend(q[:0], table[:0], n[:0], window=window, sinks=sinks).shape == (0, 4, dim)
    assert _lib.lib().bw_device_status() == 0


@pytest.mark.parametrize("heads,kv_heads,dim,bits", [(8, 2, 128, 4), (4, 4, 64, 8), (6, 1, 128, 2), (32, 2, 64, 4), (4, 2, 256, 8), (4, 2, 80, 4)])
def test_one_visible_token_gives_its_value(heads, kv_heads, dim, bits):
    """Of a window of one, and of a sink alone: the value, rounded once, also where it lies halfway between two results."""
    for window, sinks, dtype in ((1, 0, torch.float16), (0, 1, torch.bfloat16)):
        lengths = [1, 37, 16, 900, 33] * 8
        cache, table, n, slots = _filled(lengths, kv_heads, dim, bits, 16, window, sinks, 11)
        q = torch.randn(len(lengths), heads, dim, generator=_gen(12), device=DEV).to(dtype)
        want = cache.read(torch.cat(slots), dtype=dtype)[1].repeat_interleave(heads // kv_heads, 1)
        assert torch.equal(cache.attend(q, table, n, window=window, sinks=sinks), want)


def test_masked_rows_of_visible_pages_do_not_count():
    """Tokens before the window and behind the sinks on the same pages have the largest scores, infinite constants and NaN."""
    n, window, sinks, page = 200, 50, 5, 64
    cache = QuantizedKVCache(4, page, 2, 128, bits=8, device=DEV)
    slots = torch.arange(n, device=DEV)
    k, v = _rows((n, 2, 128), 13), _rows((n, 2, 128), 14)
    hidden = (slots >= sinks) & (slots < n - window)
    k[hidden] *= 100
    v[hidden] *= 100
    cache.append(k, v, slots)
    cache.params[0, :, 6] = math.nan
    cache.params[2, :, 10] = math.inf
    cache.params[2, :, 9, 0] = -math.inf
    q = torch.randn(1, 8, 128, generator=_gen(15), device=DEV).half()
    table = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    got = cache.attend(q, table, torch.tensor([n], dtype=torch.int32, device=DEV), window=window, sinks=sinks)
    _check(got, *_attended(cache, q, [slots[~hidden]], 128 ** -0.5))


def test_strides_scale_and_captured_steps():
    lengths = [500, 130, 16, 2000]
    cache, table, n, slots = _filled(lengths, 2, 128, 4, 16, 100, 8, 16)
    wide = torch.randn(4, 10, 256, generator=_gen(17), device=DEV).half()
    q = wide[:, 1:9, :128]
    table2 = torch.full((4, 2 * table.shape[1] + 5), -7, dtype=torch.int32, device=DEV)
    table2[:, :table.shape[1]] = table
    want, size = _attended(cache, q, slots, 0.3)
    for args in ((q, table, n), (q, table2, n), (q, table2[:, :table.shape[1]], n), (q.transpose(1, 2).contiguous().transpose(1, 2), table, n),
                 (q, table.T.contiguous().T, n.repeat_interleave(2)[::2])):
        _check(cache.attend(*args, softmax_scale=0.3, window=100, sinks=8), want, size)
    # a captured window slides with the lengths of its replay
    n2 = torch.tensor([300, 17, 0, 900], dtype=torch.int32, device=DEV)
    full, full_table, _, _ = _filled([2000] * 4, 2, 128, 4, 16, 10 ** 6, 0, 18)
    graph = torch.cuda.CUDAGraph()
    full.attend(q, full_table, n2, window=100, sinks=8)
    with torch.cuda.graph(graph):
        out = full.attend(q, full_table, n2, window=100, sinks=8)
    for step in range(3):
        n2 += torch.tensor([1, 40, 3, 350], dtype=torch.int32, device=DEV)
        graph.replay()
        rows = []
        for b, m in enumerate(n2.tolist()):
            t = _visible(m, 100, 8)
            rows.append(full_table[b].long()[t // 16] * 16 + t % 16)
        _check(out, *_attended(full, q, rows, 128 ** -0.5))
