"""Attention over the quantised cache holds its weights and queries as exactly as fp32 sums do, whatever the result's type."""
import pytest
import torch

from bitween_b200 import QuantizedKVCache
from bitween_b200.kernels import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _between(got, want, slack):
    """Rounding keeps order: a value within `slack` of `want`, rounded once, lies between the two ends' roundings."""
    return (got >= (want - slack).to(got.dtype)) & (got <= (want + slack).to(got.dtype))


@pytest.mark.parametrize("heads,kv_heads,dim,bits,lengths", [
    (4, 4, 128, 4, [24] * 48),                     # up to four heads a cache head: steps of two tiles
    (16, 4, 64, 8, [40, 9, 24, 1] * 16),
    (16, 4, 128, 2, [33] * 24),
    (12, 2, 128, 8, [24] * 32),                    # five to eight: steps of one
    (32, 2, 64, 4, [24] * 32),                     # more: two blocks of eight columns
    (4, 2, 256, 4, [24] * 24),
    (8, 2, 128, 4, [700, 30] * 20),                # shares of the line of work, and a join
    (6, 6, 80, 4, [24] * 32),                      # the general kernel
])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_weights_keep_more_bits_than_the_result(heads, kv_heads, dim, bits, lengths, dtype):
    """With scores of at most 1/2 (in powers of two) their fp32 errors are below 2^-19.5 of a weight: at most 20 truncated accumulations of products and three roundings
    of the zero point's part, 2^-23 of 1/2 each.  ex2 is good to 2^-22, a weight is held to 2^-22 (value and rest, 11 bits each) and the sums over a warp's few steps
    and the join to some 2^-23.  Numerator and denominator together: less than 2^-17.5 of sum w |v|.  (A weight of 11 bits is off by up to 2^-12.)"""
    page, batch = 16, len(lengths)
    wide = -(-max(lengths) // page)
    cache = QuantizedKVCache(batch * wide, page, kv_heads, dim, bits=bits, device=DEV)
    table = torch.randperm(batch * wide, generator=_gen(1), device=DEV).view(batch, wide)
    pos = torch.arange(wide * page, device=DEV)
    slots = table[:, pos // page] * page + pos % page
    cache.append(*(torch.randn(slots.numel(), kv_heads, dim, generator=_gen(s), device=DEV) * (0.5 + torch.rand(slots.numel(), kv_heads, 1, generator=_gen(s + 9), device=DEV))
                   for s in (2, 3)), slots.flatten())
    q = torch.randn(batch, heads, dim, generator=_gen(4), device=DEV).to(dtype)
    k, v = (x.double().view(batch, wide * page, kv_heads, dim) for x in cache.read(slots.flatten(), dtype=torch.float32))
    span = cache.params[..., 0].float().amax() * (2 ** bits - 1)
    alpha = 0.5 / (1.4427 * float(span * q.float().abs().sum(-1).amax()))
    got = cache.attend(q, table.to(torch.int32), torch.tensor(lengths, dtype=torch.int32, device=DEV), softmax_scale=alpha)
    group = heads // kv_heads
    score = torch.einsum("bhgd,bthd->bhgt", q.double().view(batch, kv_heads, group, dim), k) * alpha
    live = pos[None] < torch.tensor(lengths, device=DEV)[:, None]
    w = torch.softmax(score.masked_fill(~live[:, None, None], -torch.inf), -1)
    want = torch.einsum("bhgt,bthd->bhgd", w, v).view(q.shape)
    size = torch.einsum("bhgt,bthd->bhgd", w, v.abs()).view(q.shape)
    ok = _between(got, want, 2.0 ** -17.5 * size)
    bad = int((~ok).sum())
    assert bad == 0, f"{bad} of {ok.numel()}"
    assert _lib.lib().bw_device_status() == 0


@pytest.mark.parametrize("dim,heads", [(64, 2), (128, 8), (256, 2), (128, 16), (80, 2)])
def test_bf16_queries_of_a_wide_range(dim, heads):
    """One element 2^22 times the others, where every key is zero: the others keep all their bits.  (Rows that are not negative have a zero point of 0: nothing
    cancels, and scores have the fp32 errors of the small elements' products alone.)"""
    batch, n = 8, 40
    cache = QuantizedKVCache(batch * 3, 16, 1, dim, bits=8, device=DEV)
    slots = torch.arange(batch * 48, device=DEV)
    k = torch.rand(batch * 48, 1, dim, generator=_gen(11), device=DEV)
    k[..., 0] = 0
    cache.append(k, torch.randn(k.shape, generator=_gen(12), device=DEV), slots)
    q = torch.randn(batch, heads, dim, generator=_gen(13), device=DEV) * 2.0 ** -12
    q[..., 0] = 2.0 ** 10
    q = q.bfloat16()
    table = torch.arange(batch * 3, dtype=torch.int32, device=DEV).view(batch, 3)
    alpha = 2.0 ** 12 * dim ** -0.5
    got = cache.attend(q, table, torch.full((batch,), n, dtype=torch.int32, device=DEV), softmax_scale=alpha)
    kd, vd = (x.double().view(batch, 48, dim)[:, :n] for x in cache.read(slots, dtype=torch.float32))
    w = torch.softmax(torch.einsum("bhd,btd->bht", q.double(), kd) * alpha, -1)
    want, size = torch.einsum("bht,btd->bhd", w, vd), torch.einsum("bht,btd->bhd", w, vd.abs())
    # scores of sums of up to 256 products of about 1/2, 2^-23 of their absolute sum (up to 14) a block of 16: 2^-15; twice, for numerator and denominator
    ok = _between(got, want, 2.0 ** -14 * size)
    bad = int((~ok).sum())
    assert bad == 0, f"{bad} of {ok.numel()}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("below", [25.5, 28.5])
def test_many_tokens_far_below_one_that_dominates(dtype, below):
    """4095 tokens at 2^-25.5 of a dominant one: they are all of the result where the dominant token's value is zero.  64 sequences of the same pages, so that a
    warp has some hundred of the tokens beside the dominant one."""
    n, dim, batch, kv_heads = 4096, 64, 64, 8
    cache = QuantizedKVCache(n // 16, 16, kv_heads, dim, bits=8, device=DEV)
    k, v = torch.zeros(n, kv_heads, dim, device=DEV), torch.ones(n, kv_heads, dim, device=DEV)
    v[..., 0] = 0
    for h in range(kv_heads):
        k[500 * h + 77, h, 0] = 1
        v[500 * h + 77, h] = 0
        v[500 * h + 77, h, 0] = 1
    cache.append(k, v, torch.arange(n, device=DEV))
    kd, vd = (x.double().transpose(0, 1) for x in cache.read(torch.arange(n, device=DEV), dtype=torch.float32))
    q = torch.zeros(batch, 4 * kv_heads, dim, device=DEV)
    q[..., 0] = 1
    alpha = below * 0.6931471805599453 / float(kd.amax())
    table = torch.arange(n // 16, dtype=torch.int32, device=DEV)[None].expand(batch, -1)
    got = cache.attend(q.to(dtype), table, torch.full((batch,), n, dtype=torch.int32, device=DEV), softmax_scale=alpha)
    w = torch.softmax(kd[..., 0] * alpha, -1)[:, None]
    want, size = ((w @ x).expand(-1, 4, -1).reshape(1, 4 * kv_heads, dim).expand(batch, -1, -1) for x in (vd, vd.abs()))
    # The largest weight times its scale is 2^12 at least where it is reached, fp16's smallest step 2^-24: a weight counts to within 2^-37 of the largest, 4096 of them to 2^-25;
    # 2^-17 for the score (30, 2^-24 of it a rounding) and the sums.
    slack = 2.0 ** -17 * size + 2.0 ** -25
    ok = _between(got, want, slack + (2.0 ** -25 if dtype == torch.float16 else 0))
    bad = int((~ok).sum())
    assert bad == 0, (bad, got[0, 0, :3].tolist(), want[0, 0, :3].tolist())


@pytest.mark.parametrize("heads,kv_heads,dim,bits,batch,wide", [(8, 2, 128, 4, 40, 1), (4, 4, 64, 8, 40, 1), (6, 1, 128, 2, 40, 1), (32, 2, 64, 4, 20, 1), (4, 2, 256, 8, 20, 1), (8, 2, 128, 4, 60, 400),
                                                                 (4, 2, 80, 4, 20, 1)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_sequence_of_one_token_gives_its_value(heads, kv_heads, dim, bits, batch, wide, dtype):
    """The weight is 1: what comes out is the value, rounded once, also where it lies halfway between two results."""
    cache = QuantizedKVCache(batch * wide, 16, kv_heads, dim, bits=bits, device=DEV)
    table = torch.arange(batch * wide, dtype=torch.int32, device=DEV).view(batch, wide)
    slots = table[:, 0].long() * 16
    cache.append(torch.randn(batch, kv_heads, dim, generator=_gen(31), device=DEV), torch.randn(batch, kv_heads, dim, generator=_gen(32), device=DEV), slots)
    lengths = torch.ones(batch, dtype=torch.int32, device=DEV)
    if wide > 1:
        lengths[0] = 16 * wide                          # (rows of zeros behind the first: shares of the line of work)
    q = torch.randn(batch, heads, dim, generator=_gen(33), device=DEV).to(dtype)
    want = cache.read(slots, dtype=dtype)[1].repeat_interleave(heads // kv_heads, 1)
    got = cache.attend(q, table, lengths)
    assert torch.equal(got[1:], want[1:]) and (wide > 1 or torch.equal(got[0], want[0]))
    assert _lib.last_kernel() == ("kv_attend_general_kernel" if dim == 80 else "kv_attend_join_kernel" if wide > 1 else "kv_attend_kernel")
    bad = torch.randn(1, kv_heads, dim, device=DEV)
    bad[..., 3] = torch.nan
    cache.append(bad, bad, slots[1:2])
    got = cache.attend(q, table, lengths)
    assert bool(got[1].isnan().all()) and torch.equal(got[2:], want[2:])
