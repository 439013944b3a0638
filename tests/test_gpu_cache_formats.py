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
