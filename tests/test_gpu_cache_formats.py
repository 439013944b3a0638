"""Caches that other quantizers have filled: `from_tensors` takes any scales and zero points, and a row stands for scale * (code - zero_point)."""
import pytest
import torch

from bitween_b200 import QuantizedKVCache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _adopted(pages, heads, dim, bits, page, zeros):
    """(cache, keys, values) of random codes; `zeros`: what the zero points are like."""
    g, q = _gen(1), 2 ** bits - 1
    words = [torch.randint(-2 ** 31, 2 ** 31, (pages, heads, page, dim * bits // 32), generator=g, device=DEV).to(torch.int32) for _ in range(2)]
    params = torch.empty(pages, heads, page, 4, device=DEV)
    params[..., 0::2] = (0.5 + torch.rand(params[..., 0::2].shape, generator=g, device=DEV)) * 4 / q
    u = torch.rand(params[..., 1::2].shape, generator=g, device=DEV)
    params[..., 1::2] = {"fractions": u * q, "outside": u * 9 * q - 4 * q, "7.3 and 1.5": torch.where(u < 0.5, 7.3, 1.5), "signs": u * q, "far": torch.round(1000 + 3000 * u)}[zeros]
    if zeros == "signs":
        params[..., 0::2] *= torch.where(torch.rand(params[..., 0::2].shape, generator=g, device=DEV) < 0.5, -1.0, 1.0)
    params = params.half()
    shifts = torch.arange(0, 32, bits, device=DEV)
    rows = []
    for w, at in ((words[0], 0), (words[1], 2)):
        code = ((w.long()[..., None] >> shifts) & q).flatten(-2).double()
        p = params.double()
        rows.append((p[..., at, None] * (code - p[..., at + 1, None])).transpose(1, 2).reshape(pages * page, heads, dim))
    return QuantizedKVCache.from_tensors(*words, params, bits), *rows


ZEROS = ["fractions", "outside", "7.3 and 1.5", "signs", "far"]


@pytest.mark.parametrize("zeros", ZEROS)
@pytest.mark.parametrize("bits", [2, 4, 8])
@pytest.mark.parametrize("dim", [80, 128])
def test_read_gives_what_a_row_stands_for(zeros, bits, dim):
    cache, k, v = _adopted(3, 2, dim, bits, 16, zeros)
    slots = torch.randperm(48, generator=_gen(2), device=DEV)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for got, want in zip(cache.read(slots, dtype=dtype), (k, v)):
            assert torch.equal(got, want[slots].float().to(dtype))


@pytest.mark.parametrize("zeros", ZEROS)
@pytest.mark.parametrize("bits", [2, 4, 8])
@pytest.mark.parametrize("heads,kv_heads,dim,page,lengths", [
    (8, 2, 128, 16, [300, 1, 40, 0, 17]), (6, 1, 64, 32, [300, 55]), (16, 1, 128, 16, [100, 31]), (4, 2, 256, 16, [200, 3]),
    (8, 2, 128, 16, [3000, 17, 900]), (4, 2, 80, 16, [100, 9]), (4, 2, 64, 7, [100, 9])])
def test_attend_takes_any_scale_and_zero_point(zeros, bits, heads, kv_heads, dim, page, lengths):
    """Tiled kernel (clusters, shares) and general kernel.  Scores of at most 1/2 plus what the zero point adds; values' sums have the bound of `test_gpu_kv_cache.py`."""
    batch, wide = len(lengths), -(-max(lengths) // page)
    cache, k, v = _adopted(batch * wide + 1, kv_heads, dim, bits, page, zeros)
    table = torch.randperm(batch * wide + 1, generator=_gen(3), device=DEV)[:batch * wide].view(batch, wide)
    group = heads // kv_heads
    for dtype in (torch.float16, torch.bfloat16):
        q = torch.randn(batch, heads, dim, generator=_gen(4), device=DEV).to(dtype)
        alpha = 0.5 / float(q.float().abs().sum(-1).amax() * 6)
        got = cache.attend(q, table.to(torch.int32), torch.tensor(lengths, dtype=torch.int32, device=DEV), softmax_scale=alpha)
        # fp32 errors of scores: 20 accumulations and roundings, 2^-23 of alpha * sum |q| * scale * (code + |zero point|) each
        reach = float((cache.params[..., 0].float().abs() * (2 ** bits + cache.params[..., 1].float().abs())).amax()) / 12
        for b, n in enumerate(lengths):
            if n == 0:
                assert bool((got[b] == 0).all())
                continue
            pos = torch.arange(n, device=DEV)
            at = table[b, pos // page] * page + pos % page
            kd, vd = k[at].repeat_interleave(group, 1), v[at].repeat_interleave(group, 1)
            w = torch.softmax(torch.einsum("hd,thd->ht", q[b].double(), kd) * alpha, -1)
            want, size = torch.einsum("ht,thd->hd", w, vd), torch.einsum("ht,thd->hd", w, vd.abs())
            half = torch.finfo(dtype).eps / 2
            err = (got[b].double() - want).abs()
            assert bool((err <= half * want.abs() + (2.0 ** -11 + 2 * 20 * 2.0 ** -23 * reach) * size + 1e-6).all()), float(err.max())
