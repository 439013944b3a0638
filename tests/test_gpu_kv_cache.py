"""The quantised key-value cache: rows written and read back bit for bit, attention against 64-bit sums."""
import math
import threading

import pytest
import torch

from bitween_b200 import QuantizedKVCache, dequantize_rtn
from bitween_b200.kernels import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rows(shape, seed, dtype):
    g = _gen(seed)
    x = torch.randn(shape, generator=g, device=DEV) * (0.5 + torch.rand(shape[-1], generator=g, device=DEV))
    return (x + 0.3 * torch.randn(shape[-1], generator=g, device=DEV)).to(dtype)


def quantised(x, bits):
    """(codes, scale, zero) of the rows of x by the steps of the definition, each rounded once in fp32."""
    x, most = x.float(), torch.tensor(float(2 ** bits - 1), device=x.device)
    lo, hi = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
    span = (hi - lo) / most
    s = span.half()
    s = torch.where(s.float() < span, (s.view(torch.int16) + 1).view(torch.float16), s).clamp(min=2.0 ** -24)
    sf = s.float()
    z = torch.round(-lo / sf)
    return torch.clamp(torch.round(x / sf[..., None] + z[..., None]), 0, 2 ** bits - 1), s, z


def stands_for(x, bits):
    c, s, z = quantised(x, bits)
    return s.double()[..., None] * (c.double() - z.double()[..., None])


@pytest.mark.parametrize("bits", [2, 4, 8])
@pytest.mark.parametrize("dim", [16, 64, 80, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_rows_are_written_and_read_back(bits, dim, dtype):
    tokens, heads, page = 37, 3, 16
    cache = QuantizedKVCache(5, page, heads, dim, bits=bits, device=DEV)
    cache.k_codes.fill_(-1)
    cache.v_codes.fill_(-1)
    cache.params.fill_(7)
    fused = _rows((tokens, 3 * heads, dim), 1, dtype)            # q, k, v in one tensor: strided rows
    k, v = fused[:, heads:2 * heads], fused[:, 2 * heads:]
    k[3] = 0
    k[4] = k[4].abs() + 1
    k[5] = -k[5].abs() - 1
    k[6] *= 1e-6
    v[7] *= 1e-3
    slots = torch.randperm(5 * page, generator=_gen(2), device=DEV)[:tokens]
    slots[11], slots[12] = -1, 5 * page                           # skipped
    cache.append(k, v, slots)
    names = torch.ones(5 * page, dtype=torch.bool, device=DEV)
    live = (slots >= 0) & (slots < 5 * page)
    names[slots[live]] = False
    rest = names.view(5, page)
    for codes, params, x in ((cache.k_codes, cache.params[..., :2], k), (cache.v_codes, cache.params[..., 2:], v)):
        # rows that were not named are left as they were
        assert bool((codes.transpose(1, 2)[rest] == -1).all()) and bool((params.transpose(1, 2)[rest] == 7).all())
        c, s, z = quantised(x[live], bits)
        at, off = slots[live] // page, slots[live] % page
        assert torch.equal(params[at, :, off, 0], s) and torch.equal(params[at, :, off, 1].float(), z)
        # the packed format of weights: dequantize_rtn reads it
        n = codes.numel() * 32 // bits // dim
        w = dequantize_rtn(codes.view(n, -1), torch.ones(n, 1, device=DEV), torch.zeros(n, 1, device=DEV), dim, bits=bits)
        assert torch.equal(w.view(5, heads, page, dim)[at, :, off], c)
    for out in (torch.float16, torch.bfloat16, torch.float32):
        rk, rv = cache.read(slots, dtype=out)
        for got, x in ((rk, k), (rv, v)):
            want = stands_for(x, bits)
            want[~live] = 0
            assert torch.equal(got, want.float().to(out))
    # half a step of rounding, the step at most a rounding up of fp16 above (hi - lo) / Q; the rest are fp32 roundings of codes up to 255
    step = cache.read(slots, dtype=torch.float32)[0][live].double() - k[live].double()
    s = quantised(k[live], bits)[1].double()[..., None]
    assert bool((step.abs() <= s * (0.5 + 2.0 ** -14)).all())


def test_rows_with_nan_infinity_or_too_large_read_back_as_nan():
    cache = QuantizedKVCache(1, 16, 2, 64, bits=4, device=DEV)
    k = torch.randn(6, 2, 64, device=DEV)
    v = torch.randn(6, 2, 64, device=DEV)
    k[0, 0, 5] = math.nan
    k[1, 1, 6] = math.inf
    v[2, 0, 7] = -math.inf
    v[3, 1, 8] = 3e38
    v[4, 0, 9] = -3e38
    v[4, 0, 10] = 3e38
    cache.append(k, v, torch.arange(6, device=DEV))
    rk, rv = cache.read(torch.arange(6, device=DEV), dtype=torch.float32)
    bad_k = torch.zeros(6, 2, dtype=torch.bool, device=DEV)
    bad_v = bad_k.clone()
    bad_k[0, 0] = bad_k[1, 1] = True
    bad_v[2, 0] = bad_v[3, 1] = bad_v[4, 0] = True
    for got, x, bad in ((rk, k, bad_k), (rv, v, bad_v)):
        assert bool(got[bad].isnan().all())
        assert torch.equal(got[~bad], stands_for(x[~bad], 4).float())


def _filled(lengths, heads, dim, bits, page, seed, dtype=torch.float16, spare=2):
    """A cache with sequences of these lengths on scattered pages; every row that no sequence holds reads as NaN."""
    wide = max(1, -(-max(lengths) // page))
    pages = len(lengths) * wide + spare
    cache = QuantizedKVCache(pages, page, heads, dim, bits=bits, device=DEV)
    cache.params.fill_(math.nan)
    table = torch.randperm(pages, generator=_gen(seed), device=DEV)[:len(lengths) * wide].view(len(lengths), wide)
    pos = torch.arange(wide * page, device=DEV)
    slots = table[:, pos // page] * page + pos % page
    held = pos[None] < torch.tensor(lengths, device=DEV)[:, None]
    for part in slots[held].split(1 << 16):
        shape = (part.numel(), heads, dim)
        cache.append(_rows(shape, seed + 1, dtype), _rows(shape, seed + 2, dtype), part)
    return cache, table.to(torch.int32), torch.tensor(lengths, dtype=torch.int32, device=DEV), slots


def _attended(cache, q, slots, lengths, alpha):
    """(outputs, sums of w |v|) in 64 bits."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(out)
    group = q.shape[1] // cache.num_kv_heads
    for b, n in enumerate(lengths):
        if n <= 0:
            continue
        k, v = (x.double() for x in cache.read(slots[b, :n].contiguous(), dtype=torch.float32))
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        w = torch.softmax(torch.einsum("hd,thd->ht", q[b].double(), k) * alpha, -1)
        out[b] = torch.einsum("ht,thd->hd", w, v)
        size[b] = torch.einsum("ht,thd->hd", w, v.abs())
    return out, size


def _check(got, want, size):
    """The result's own rounding, and weights held in fp16 (2^-11 of each); the scores' fp32 errors are far below that."""
    half = torch.finfo(got.dtype).eps / 2
    assert bool(((got.double() - want).abs() <= half * want.abs() + 2.0 ** -11 * size + 1e-6).all())


@pytest.mark.parametrize("lengths,heads,kv_heads,dim,bits,page", [
    ([1], 1, 1, 64, 8, 16),
    ([49], 12, 12, 64, 8, 16),
    ([0, 1, 15, 16, 17, 33, 0], 8, 2, 128, 4, 16),
    ([300, 5, 129], 10, 2, 128, 2, 48),
    ([0, 0], 4, 4, 128, 4, 16),
    ([700, 64, 1000], 16, 2, 128, 8, 64),
    ([257, 31], 32, 2, 256, 4, 32),
    ([511], 24, 2, 64, 2, 16),
    ([100, 1], 7, 1, 256, 8, 16),
    ([90, 3], 34, 1, 128, 4, 16),
    ([2100, 40, 801], 14, 2, 128, 4, 16),
    ([4099], 8, 1, 256, 2, 16),
    ([5000], 5, 1, 64, 4, 16),
    ([40, 9, 0], 6, 3, 80, 4, 16),        # a head size and a page size of the general kernel
    ([100, 33], 4, 2, 128, 8, 7),
    ([20011], 4, 2, 128, 4, 16),
])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend(lengths, heads, kv_heads, dim, bits, page, dtype):
    cache, table, n, slots = _filled(lengths, kv_heads, dim, bits, page, 3)
    q = torch.randn(len(lengths), heads, dim, generator=_gen(4), device=DEV).to(dtype)
    got = cache.attend(q, table, n)
    assert got.dtype == dtype and got.shape == q.shape
    want, size = _attended(cache, q, slots, lengths, dim ** -0.5)
    _check(got, want, size)
    assert torch.equal(got, cache.attend(q, table, n))             # no sum depends on the order of arrival
    assert _lib.lib().bw_device_status() == 0


@pytest.mark.parametrize("scale", [1e-3, 3.0, 200.0, 3e4])
def test_attend_queries_and_values_far_from_one(scale):
    lengths = [333, 40]
    cache, table, n, slots = _filled(lengths, 2, 128, 4, 16, 5)
    cache.params[..., 2] *= 2.0 ** -9                               # values of about 1e-3: small steps in fp16
    q = (torch.randn(2, 8, 128, generator=_gen(6), device=DEV) * scale).clamp(-6e4, 6e4)
    for dtype in (torch.float16, torch.bfloat16):
        want, size = _attended(cache, q.to(dtype), slots, lengths, 128 ** -0.5)
        got = cache.attend(q.to(dtype), table, n)
        # scores of up to alpha |q| |k| ~ 10 * scale have fp32 errors of 2^-20 of that: the weights' relative error
        half = torch.finfo(dtype).eps / 2
        assert bool(((got.double() - want).abs() <= half * want.abs() + (2.0 ** -11 + 2.0 ** -20 * 12 * scale) * size + 2.0 ** -24).all())


def test_attend_takes_scores_that_rise_and_fall():
    """Keys that grow along the sequence move the running maximum many times over, downwards and upwards."""
    lengths = [3000, 2999]
    cache, table, n, slots = _filled(lengths, 2, 64, 8, 16, 7)
    ramp = torch.linspace(0.01, 12, 3000, device=DEV)
    for b, order in ((0, ramp), (1, ramp.flip(0))):
        t = slots[b, :lengths[b]].contiguous()
        k = _rows((t.numel(), 2, 64), 8, torch.float32) * order[:t.numel(), None, None]
        cache.append(k, _rows(k.shape, 9, torch.float32), t)
    q = torch.randn(2, 4, 64, generator=_gen(10), device=DEV).half()
    want, size = _attended(cache, q, slots, lengths, 1.0)
    # scores of up to 12 * 64 have fp32 errors of 2^-20 of that
    got = cache.attend(q, table, n, softmax_scale=1.0)
    assert bool(((got.double() - want).abs() <= 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -20 * 770) * size + 1e-6).all())


def test_attend_strides_and_scale():
    lengths = [77, 130, 16]
    cache, table, n, slots = _filled(lengths, 2, 128, 4, 16, 11)
    wide = torch.randn(3, 10, 256, generator=_gen(12), device=DEV).half()
    q = wide[:, 1:9, :128]
    table2 = torch.full((3, 2 * table.shape[1] + 5), -7, dtype=torch.int32, device=DEV)
    table2[:, :table.shape[1]] = table
    want, size = _attended(cache, q, slots, lengths, 0.3)
    _check(cache.attend(q, table2[:, :table.shape[1]], n, softmax_scale=0.3), want, size)
    _check(cache.attend(q, table2, n, softmax_scale=0.3), want, size)              # pages beyond the lengths are not looked at
    _check(cache.attend(q.transpose(1, 2).contiguous().transpose(1, 2), table, n, softmax_scale=0.3), want, size)
    odd = wide.flatten()[1:1 + 3 * 8 * 128].view(3, 8, 128)                         # rows off a 16-byte boundary
    want, size = _attended(cache, odd, slots, lengths, 0.3)
    _check(cache.attend(odd, table, n, softmax_scale=0.3), want, size)


@pytest.mark.parametrize("dim,page", [(128, 16), (80, 16)])
def test_attend_bad_pages_and_lengths_are_loud(dim, page):
    lengths = [40, 40, 40, 200, 40, 7]
    cache, table, n, slots = _filled(lengths, 2, dim, 4, page, 13)
    q = torch.randn(6, 4, dim, generator=_gen(14), device=DEV).half()
    want, size = _attended(cache, q, slots, lengths, dim ** -0.5)
    table[1, 2] = cache.num_pages
    table[2, 0] = -1
    table[5, 1:] = 2 ** 31 - 1                                       # not reached: 7 tokens
    n[0], n[4] = -3, 13 * 16 + 1
    got = cache.attend(q, table, n)
    assert bool((got[0] == 0).all())
    assert bool(got[[1, 2, 4]].isnan().all())
    _check(got[[3, 5]], want[[3, 5]], size[[3, 5]])
    empty = cache.attend(q, table[:, :0], torch.zeros_like(n))
    assert bool((empty == 0).all())
    assert bool(cache.attend(q, table[:, :0], n)[1:].isnan().all())
    assert cache.attend(q[:0], table[:0], n[:0]).shape == (0, 4, dim)
    assert _lib.lib().bw_device_status() == 0


def test_a_nan_row_within_the_length_reaches_only_its_own_head():
    lengths = [100, 60]
    cache, table, n, slots = _filled(lengths, 2, 128, 4, 16, 15)
    bad = torch.randn(1, 2, 128, device=DEV)
    bad[0, 1, 3] = math.inf
    cache.append(torch.randn(1, 2, 128, device=DEV), bad, slots[0, 50:51].contiguous())
    q = torch.randn(2, 4, 128, generator=_gen(16), device=DEV).half()
    got = cache.attend(q, table, n)
    assert bool(got[0, 2:].isnan().all()) and bool(got[0, :2].isfinite().all()) and bool(got[1].isfinite().all())


def test_attend_shared_pages_and_offsets_past_32_bits():
    """Two sequences that share a prefix, on pages whose rows lie more than 2^31 words into the cache."""
    heads, dim, bits, page = 8, 256, 8, 64
    pages = (1 << 31) // (heads * page * dim * bits // 32) + 9      # 2^31 words of codes, 8 GB each for keys and values
    cache = QuantizedKVCache(pages, page, heads, dim, bits=bits, device=DEV)
    table = torch.tensor([[pages - 1, pages - 2, pages - 4], [pages - 1, pages - 2, pages - 3]], dtype=torch.int32, device=DEV)
    pos = torch.arange(3 * page, device=DEV)
    slots = table.long()[:, pos // page] * page + pos % page
    for b, s in ((0, 1), (1, 2)):
        shape = (2 * page if b == 0 else page, heads, dim)
        t = slots[0, :2 * page] if b == 0 else slots[1, 2 * page:]
        cache.append(_rows(shape, s, torch.float16), _rows(shape, s + 5, torch.float16), t.contiguous())
    cache.append(_rows((page, heads, dim), 3, torch.float16), _rows((page, heads, dim), 4, torch.float16), slots[0, 2 * page:].contiguous())
    lengths = [150, 190]
    q = torch.randn(2, 16, dim, generator=_gen(17), device=DEV).half()
    want, size = _attended(cache, q, slots, lengths, dim ** -0.5)
    _check(cache.attend(q, table, torch.tensor(lengths, dtype=torch.int32, device=DEV)), want, size)


def test_graphs_streams_and_threads():
    lengths = [3000, 17, 801, 0]
    cache, table, n, slots = _filled(lengths, 4, 128, 4, 16, 18)
    qs = [torch.randn(4, 8, 128, generator=_gen(20 + i), device=DEV).half() for i in range(3)]
    want = [cache.attend(q, table, n) for q in qs]
    graphs, outs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([cache.attend(q, table, n) for _ in range(8)])
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for out in outs:
            for y in out:
                y.zero_()
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        eager = [cache.attend(q, table, n) for q in qs]
        torch.cuda.synchronize()
        for out, y, ref in zip(outs, eager, want):
            assert torch.equal(y, ref) and all(torch.equal(o, ref) for o in out)
    wrong = []

    def work(i):
        for _ in range(50):
            if not torch.equal(cache.attend(qs[i], table, n), want[i]):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_captured_decode_step_takes_the_lengths_of_its_replay():
    """append and attend in one graph: tokens, slots and lengths are read when it is replayed."""
    lengths = [100, 37]
    cache, table, n, slots = _filled([160, 160], 2, 128, 8, 16, 30)
    n.copy_(torch.tensor(lengths))
    k, v = _rows((2, 2, 128), 31, torch.float16), _rows((2, 2, 128), 32, torch.float16)
    q = torch.randn(2, 8, 128, generator=_gen(33), device=DEV).half()
    at = torch.stack([slots[b, m] for b, m in enumerate(lengths)])
    cache.attend(q, table, n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(k, v, at)
        n += 1
        out = cache.attend(q, table, n)
    for step in range(4):
        k.copy_(_rows((2, 2, 128), 40 + step, torch.float16))
        v.copy_(_rows((2, 2, 128), 50 + step, torch.float16))
        at.copy_(torch.stack([slots[b, m + step] for b, m in enumerate(lengths)]))
        graph.replay()
        want, size = _attended(cache, q, slots, [m + step + 1 for m in lengths], 128 ** -0.5)
        _check(out, want, size)
        assert torch.equal(cache.read(at, dtype=torch.float32)[1].double(), stands_for(v, 8))
