"""Rank values of the adapters are held as exactly as fp32 sums are, whatever their range and the result's type."""
import pytest
import torch

from bitween_b200 import adapter_matmul
from bitween_b200.kernels import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rand(shape, seed):
    return 0.5 + torch.rand(shape, generator=_gen(seed), device=DEV)


def _outside(got, want, slack):
    """How many values are not a value within `slack` of `want` rounded once (rounding keeps order)."""
    return int((~((got >= (want - slack).to(got.dtype)) & (got <= (want + slack).to(got.dtype)))).sum())


# A result that is ONE product of a rank value, of positive numbers: fp32 sums of 64 products (4 blocks truncated at 2^-23 of the sum, in parts that are added up: 2^-20.5),
# the factor and the product's parts (2^-22 in all).  (A rank value of 16 bits is off by up to 2^-17.)
ONE_PRODUCT = 2.0 ** -19.5


@pytest.mark.parametrize("M,n,r,N", [(40, 3, 8, 4096), (300, 3, 16, 1024), (300, 2, 32, 1024), (700, 1, 64, 256), (2100, 1, 64, 8200), (2100, 1, 128, 8200), (700, 9, 128, 256), (61, 24, 4, 512)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_results_hold_more_than_sixteen_bits_of_a_rank_value(M, n, r, N, dtype):
    """y and dx, in which one rank of each adapter is not zero."""
    K = 64
    index = torch.randint(0, n, (M,), generator=_gen(1), device=DEV).sort().values.to(torch.int32)
    x, down, up, grad = (_rand(s, i + 2).to(dtype) for i, s in enumerate(((M, K), (n, r, K), (n, r, N), (M, N))))
    keep = torch.arange(r, device=DEV) == r - 3
    up = torch.where(keep[:, None], up, 0)
    y = adapter_matmul(x, down, up, index)
    h = torch.einsum("tk,trk->tr", x.double(), down.double()[index.long()])
    want = h[:, r - 3, None] * up.double()[index.long(), r - 3]
    bad = _outside(y, want, ONE_PRODUCT * want)
    assert bad == 0, f"{bad} of {want.numel()}"
    # backward, with the sides of the bank exchanged: dh is a sum of 64 products
    x2 = grad.clone().requires_grad_()
    y2 = adapter_matmul(x2, up, down, index)
    (dx,) = torch.autograd.grad(y2, (x2,), x)
    bad = _outside(dx, want, ONE_PRODUCT * want)
    assert bad == 0, f"{bad} of {want.numel()}"
    assert _lib.lib().bw_device_status() == 0


@pytest.mark.parametrize("M,n,r,N", [(40, 2, 8, 1024), (100, 1, 16, 2048), (100, 3, 32, 2048), (100, 1, 64, 1024), (700, 1, 64, 2048), (2100, 1, 32, 2048), (700, 1, 128, 1032), (40, 1, 5, 256)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradients_of_banks_hold_more_than_sixteen_bits_of_a_rank_value(M, n, r, N, dtype):
    """d up and d down of one token whose gradient is not zero."""
    K = 64
    index = torch.zeros(M, dtype=torch.int32, device=DEV)
    x, down, up, dy = (_rand(s, i + 12).to(dtype) for i, s in enumerate(((M, K), (n, r, K), (n, r, N), (N,))))
    t = M // 2 + 1
    grad = torch.zeros(M, N, dtype=dtype, device=DEV)
    grad[t] = dy
    leaf = up.clone().requires_grad_()
    (dup,) = torch.autograd.grad(adapter_matmul(x, down, leaf, index), (leaf,), grad)
    want = (x[t].double() @ down[0].double().T)[:, None] * dy.double()
    bad = _outside(dup[0], want, ONE_PRODUCT * want)
    assert bad == 0, f"{bad} of {want.numel()}"
    assert bool((dup[1:] == 0).all())
    # d down: dh of 64 products, x of N columns
    wide = torch.zeros(M, N, dtype=dtype, device=DEV)
    wide[t] = dy
    leaf = up.clone().requires_grad_()
    g2 = torch.zeros(M, K, dtype=dtype, device=DEV)
    g2[t] = x[t]
    (ddown,) = torch.autograd.grad(adapter_matmul(wide, leaf, down, index), (leaf,), g2)
    bad = _outside(ddown[0], want, ONE_PRODUCT * want)
    assert bad == 0, f"{bad} of {want.numel()}"
    assert _lib.lib().bw_device_status() == 0


def _check(got, want, size, more=0.0):
    """The bound of test_gpu_adapters.py: within 2^-12 of the absolute products, rounded once."""
    slack = 2.0 ** -12 * size + (2.0 ** -24 if got.dtype == torch.float16 else 1e-30) + more
    bad = _outside(got, want, slack)
    assert bad == 0, f"{bad} of {want.numel()}"


@pytest.mark.parametrize("M,r,N", [(40, 16, 512), (300, 32, 512), (1100, 64, 1024), (1100, 64, 8200), (300, 64, 256)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_ranks_of_very_different_sizes(M, r, N, dtype):
    """Ranks down to 2^-20 of the largest: each one's gradient, and a y in which small rows of `down` meet large rows of `up`."""
    K = 128
    index = torch.zeros(M, dtype=torch.int32, device=DEV)
    size = 2.0 ** (-20.0 * torch.arange(r, device=DEV) / (r - 1))
    x = (torch.randn(M, K, generator=_gen(21), device=DEV) * 256).to(dtype)
    down = (torch.randn(1, r, K, generator=_gen(22), device=DEV) * size[:, None] * 4).to(dtype)
    up = (torch.randn(1, r, N, generator=_gen(23), device=DEV) / size[:, None] * 2.0 ** -9).to(dtype)
    grad = (torch.randn(M, N, generator=_gen(24), device=DEV) * 2.0 ** -4).to(dtype)
    leaves = [t.requires_grad_() for t in (x, down, up)]
    y = adapter_matmul(*leaves, index)
    dx, ddown, dup = torch.autograd.grad(y, leaves, grad)
    xd, dd, ud, gd = (t.detach().double() for t in (x, down[0], up[0], grad))
    h, ha = xd @ dd.T, xd.abs() @ dd.T.abs()
    dh, dha = gd @ ud.T, gd.abs() @ ud.T.abs()
    _check(y.detach(), h @ ud, ha @ ud.abs())
    _check(dup[0], h.T @ gd, ha.T @ gd.abs())
    _check(dx, dh @ dd, dha @ dd.abs())
    _check(ddown[0], dh.T @ xd, dha.T @ xd.abs())


@pytest.mark.parametrize("M,r,N", [(64, 16, 512), (300, 32, 512), (300, 64, 256), (1100, 64, 1024), (2100, 32, 1024)])
@pytest.mark.parametrize("below", [10, 16, 22, 30])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tokens_whose_gradients_are_far_below_the_largest(M, r, N, below, dtype):
    """Columns of x in which only tokens with small gradients are not zero: their sums keep their precision.

    fp16 rank values enter these sums as multiples of one power of two, by which the largest row's largest lies in [2^14, 2^15): value and rest are each rounded by at most
    2^-25 there, which is 2^-24 of 2^14 for both, 2^-38 of the largest.  That much of it, times the absolute sum of the other operand's column, is allowed as well (at 2^-30 it is
    seen: 2^-8 of a small row; sums in fp32 that hold the large rows would be off by 2^-24 of them)."""
    K = 64
    index = torch.zeros(M, dtype=torch.int32, device=DEV)
    small = torch.arange(M, device=DEV) % 2 == 1
    x = torch.randn(M, N, generator=_gen(31), device=DEV)
    x[~small, ::2] = 0
    x = (x * 256).to(dtype)
    # (two factors: a gradient of 2^-30 is nothing in fp16)
    grad = torch.randn(M, K, generator=_gen(32), device=DEV) * torch.where(small, 2.0 ** -(below // 2), 2.0 ** ((below + 1) // 2))[:, None] * 2.0 ** -4
    grad = grad.to(dtype)
    down = (torch.randn(1, r, N, generator=_gen(33), device=DEV) * N ** -0.5).to(dtype).requires_grad_()
    up = (torch.randn(1, r, K, generator=_gen(34), device=DEV) * 2.0 ** -4).to(dtype).requires_grad_()
    ddown, dup = torch.autograd.grad(adapter_matmul(x, down, up, index), (down, up), grad)
    gd, ud, xd, dd = (t.detach().double() for t in (grad, up[0], x, down[0]))
    dh, dha = gd @ ud.T, gd.abs() @ ud.T.abs()
    floor = 2.0 ** -38 if dtype == torch.float16 else 0.0
    _check(ddown[0], dh.T @ xd, dha.T @ xd.abs(), floor * dh.abs().max() * xd.abs().sum(0))
    # and rank values of tokens far below the largest, beside gradients that only they have
    x2 = (torch.randn(M, K, generator=_gen(35), device=DEV) * torch.where(small, 2.0 ** -(below // 2), 2.0 ** ((below + 1) // 2))[:, None] * 2.0 ** -4).to(dtype)
    g2 = x.detach()
    (dup,) = torch.autograd.grad(adapter_matmul(x2, up.detach(), down, index), (down,), g2)
    h, ha = x2.double() @ ud.T, x2.double().abs() @ ud.T.abs()
    _check(dup[0], h.T @ g2.double(), ha.T @ g2.double().abs(), floor * h.abs().max() * g2.double().abs().sum(0))


@pytest.mark.parametrize("r", [1, 4, 12])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_long_sums_of_the_general_kernels(r, dtype):
    """A product of 1 and 2^17 - 1 of 2^-25: one running fp32 sum would stay at 1, off by 2^-8."""
    M, K, N = 1 << 17, 8, 8
    index = torch.zeros(M, dtype=torch.int32, device=DEV)
    x, grad = torch.zeros(M, K, device=DEV), torch.full((M, N), 2.0 ** -13, device=DEV)
    x[:, 0] = 2.0 ** -12
    x[0, 0], grad[0] = 1, 1
    down, up = torch.zeros(1, r, K, device=DEV), torch.zeros(1, r, N, device=DEV)
    down[..., 0] = 1
    up = up.to(dtype).requires_grad_()
    (dup,) = torch.autograd.grad(adapter_matmul(x.to(dtype), down.to(dtype), up, index), (up,), grad.to(dtype))
    want = torch.full(dup.shape, 1 + (M - 1) * 2.0 ** -25, dtype=torch.float64, device=DEV)
    # blocks of fp32 sums, joined: 2^-20 at most
    assert _outside(dup, want, 2.0 ** -20 * want) == 0, (dup.flatten()[0], want.flatten()[0])


def test_infinities_stay_what_they_are_in_the_general_kernels():
    M = 200
    x, grad = torch.ones(M, 8, device=DEV).bfloat16(), torch.ones(M, 8, device=DEV).bfloat16()
    grad[10, 3], grad[150, 5] = torch.inf, -torch.inf
    up = torch.zeros(1, 3, 8, device=DEV).bfloat16().requires_grad_()
    (dup,) = torch.autograd.grad(adapter_matmul(x, torch.ones(1, 3, 8, device=DEV).bfloat16(), up, torch.zeros(M, dtype=torch.int32, device=DEV)), (up,), grad)
    want = 8.0 * grad.float().sum(0)
    assert torch.equal(dup[0].float(), want.bfloat16().float().expand(3, -1)) and float(want[3]) == torch.inf


def test_gradients_of_many_tokens_and_a_rank_that_is_no_multiple_of_eight():
    M, K, N, r = 5000, 64, 72, 4
    x, grad = (torch.randn(M, c, generator=_gen(41 + c), device=DEV).bfloat16() for c in (K, N))
    down, up = ((torch.randn(2, r, c, generator=_gen(43 + c), device=DEV) / 8).bfloat16().requires_grad_() for c in (K, N))
    index = torch.randint(-1, 2, (M,), generator=_gen(45), device=DEV).to(torch.int32)
    got = torch.autograd.grad(adapter_matmul(x, down, up, index), (down, up), grad)
    for a in range(2):
        t = index == a
        xd, gd, dd, ud = x[t].double(), grad[t].double(), down[a].detach().double(), up[a].detach().double()
        _check(got[0][a], (gd @ ud.T).T @ xd, (gd.abs() @ ud.T.abs()).T @ xd.abs())
        _check(got[1][a], (xd @ dd.T).T @ gd, (xd.abs() @ dd.T.abs()).T @ gd.abs())


# Long sums of positive products.  An MMA truncates the sum that it adds to, by up to 2^-23 of it: a bias that grows with the sum's length, where roundings to nearest mostly cancel
# (n of them, independent and of at most 2^-24 of a sum that grows evenly: a standard deviation of 2^-24 / 3 * sqrt(n)).
@pytest.mark.parametrize("M,n,r", [(40, 2, 16), (300, 2, 8), (300, 1, 64), (1100, 1, 128)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rank_values_of_long_rows(M, n, r, dtype):
    """14336 columns: 14 MMAs of a warp in a row (up to 64 tokens) or four and up to 224 fp32 additions (six deviations: 2^-19), and 15 additions of parts: 2^-18.5 in all."""
    K, N = 14336, 1024
    index = torch.randint(0, n, (M,), generator=_gen(51), device=DEV).sort().values.to(torch.int32)
    x, down, up = (_rand(s, i + 52).to(dtype) for i, s in enumerate(((M, K), (n, r, K), (n, r, N))))
    down *= 2.0 ** -10
    up = torch.where((torch.arange(r, device=DEV) == 3)[:, None], up, 0)
    want = torch.einsum("tk,tk->t", x.double(), down[:, 3].double()[index.long()])[:, None] * up[:, 3].double()[index.long()]
    bad = _outside(adapter_matmul(x, down, up, index), want, 2.0 ** -18.5 * want)
    assert bad == 0, f"{bad} of {want.numel()}"


@pytest.mark.parametrize("M,r,N,bound", [
    # tcgen05, a CTA for all tokens: 128 MMAs into each of two sums that grow evenly.  Each aligns 16 products and the sum to the largest of them and drops what lies below its
    # 24 bits: up to 17 * 2^-23 of the sum, of one sign where the products have one; 17 * 64 * 2^-23 in all.
    (4096, 64, 37888, 17 * 2.0 ** -17),
    (8192, 16, 1024, 2.0 ** -18.5),        # mma.sync: 16 tokens' products (three truncations), then up to 512 fp32 additions (six deviations: 2^-18.6)
    (8192, 8, 520, 2.0 ** -18.5),
    (480, 64, 1024, 2.0 ** -18.5)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradients_of_banks_summed_over_many_tokens(M, r, N, bound, dtype):
    K = 64
    index = torch.zeros(M, dtype=torch.int32, device=DEV)
    x, down, up, grad = (_rand(s, i + 62).to(dtype) for i, s in enumerate(((M, K), (1, r, K), (1, r, N), (M, N))))
    x *= 2.0 ** -9
    up.requires_grad_()
    (dup,) = torch.autograd.grad(adapter_matmul(x, down, up, index), (up,), grad)
    want = (x.double() @ down[0].double().T).T @ grad.double()
    bad = _outside(dup[0], want, (bound + 2.0 ** -20) * want)          # (2^-20: the rank values themselves, of 64 products)
    assert bad == 0, f"{bad} of {want.numel()}"
