"""Low-rank adapters beside a shared projection: forward and gradients against 64-bit sums."""
import math

import pytest
import torch

from bitween_b200 import AdaptedLinear, QuantizedKVCache, QuantizedLinear, adapter_matmul
from bitween_b200.kernels import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _bank(M, K, N, n, r, dtype, seed=1, order="any"):
    g = _gen(seed)
    x = torch.randn(M, K, generator=g, device=DEV).to(dtype)
    down = (torch.randn(n, r, K, generator=g, device=DEV) / math.sqrt(K)).to(dtype)
    up = (0.2 * torch.randn(n, r, N, generator=g, device=DEV)).to(dtype)
    base = torch.randn(M, N, generator=g, device=DEV).to(dtype)
    scaling = 0.5 + torch.rand(n, generator=g, device=DEV)
    index = torch.randint(-1, n, (M,), generator=g, device=DEV)
    if order == "runs":
        index = index.sort().values
    return x, down, up, index.to(torch.int32), scaling, base


def _formula(x, down, up, index, scaling, base, grad=None):
    """{name: (value, sum of the absolute products behind it)} in 64 bits, of the rows and adapters that have tokens."""
    x, down, up, f = (t.double() for t in (x, down, up, scaling))
    M, N = x.shape[0], up.shape[2]
    y = torch.zeros(M, N, dtype=torch.float64, device=DEV) if base is None else base.double()
    out = {"y": (y, torch.zeros_like(y)), "dx": (torch.zeros_like(x), torch.zeros_like(x)),
           "ddown": (torch.zeros_like(down), torch.zeros_like(down)), "dup": (torch.zeros_like(up), torch.zeros_like(up))}
    for i in range(down.shape[0]):
        t = (index == i).nonzero()[:, 0]
        h, ha = x[t] @ down[i].T, x[t].abs() @ down[i].T.abs()
        out["y"][0][t] += f[i] * (h @ up[i])
        out["y"][1][t] += f[i] * (ha @ up[i].abs())
        if grad is not None:
            dy = grad[t].double()
            dh, dha = f[i] * dy @ up[i].T, f[i] * dy.abs() @ up[i].T.abs()
            out["dx"][0][t], out["dx"][1][t] = dh @ down[i], dha @ down[i].abs()
            out["ddown"][0][i], out["ddown"][1][i] = dh.T @ x[t], dha.T @ x[t].abs()
            out["dup"][0][i], out["dup"][1][i] = f[i] * (h.T @ dy), f[i] * (ha.T @ dy.abs())
    return out


def _check(got, want, size):
    """The result is a value within 2^-12 of the absolute products from the formula's, rounded once: fp32 sums of up to 2^14 products in blocks
    of 16, truncated (2^-23 a block: 2^-13), in two passes, and rank values held as two 16-bit parts (2^-17).  Rounding keeps order, so it lies between the
    roundings of the two ends (beyond 65520 that is infinity in fp16: a difference would be undefined there)."""
    slack = 2.0 ** -12 * size + (2.0 ** -24 if got.dtype == torch.float16 else 1e-30)
    low, high = (want - slack).to(got.dtype), (want + slack).to(got.dtype)
    assert bool(((got >= low) & (got <= high)).all()), int((~((got >= low) & (got <= high))).sum())


SIZES = [
    # tokens, K, N, adapters, rank, order
    (1, 64, 64, 1, 8, "any"),
    (1, 4096, 4096, 3, 16, "any"),
    (5, 4096, 1024, 3, 16, "any"),
    (16, 512, 4160, 16, 8, "any"),
    (17, 1024, 512, 2, 64, "any"),
    (61, 2048, 1536, 24, 32, "any"),
    (64, 256, 256, 1, 128, "any"),
    (130, 1088, 960, 5, 16, "any"),
    (515, 1024, 2048, 4, 16, "runs"),
    (1000, 520, 776, 3, 24, "runs"),
    (300, 128, 8, 40, 8, "any"),
    (33, 8, 128, 2, 256, "any"),
    (7, 100, 130, 3, 5, "any"),              # nothing a multiple of eight: the general kernels
    (40, 4096, 96, 2, 1, "runs"),
    (2050, 768, 768, 2, 16, "runs"),
]


@pytest.mark.parametrize("M,K,N,n,r,order", SIZES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_forward(M, K, N, n, r, order, dtype):
    x, down, up, index, scaling, base = _bank(M, K, N, n, r, dtype, order=order)
    got = adapter_matmul(x, down, up, index, scaling=scaling, base=base)
    assert got.shape == (M, N) and got.dtype == dtype
    _check(got, *_formula(x, down, up, index, scaling, base)["y"])
    assert torch.equal(got[index < 0], base[index < 0])
    assert torch.equal(got, adapter_matmul(x, down, up, index, scaling=scaling, base=base))
    plain = adapter_matmul(x, down, up, index)
    _check(plain, *_formula(x, down, up, index, torch.ones_like(scaling), None)["y"])
    assert bool((plain[index < 0] == 0).all())
    adapter_matmul(x, down, up, index, scaling=scaling, base=base, out=base)          # in place
    assert torch.equal(got, base)
    assert _lib.lib().bw_device_status() == 0


@pytest.mark.parametrize("M,K,N,n,r,order", SIZES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradients(M, K, N, n, r, order, dtype):
    x, down, up, index, scaling, base = _bank(M, K, N, n, r, dtype, seed=2, order=order)
    leaves = [t.requires_grad_() for t in (x, down, up, base)]
    grad = torch.randn(M, N, generator=_gen(3), device=DEV).to(dtype)
    y = adapter_matmul(x, down, up, index, scaling=scaling, base=base)
    got = torch.autograd.grad(y, leaves, grad, retain_graph=True)
    want = _formula(x.detach(), down.detach(), up.detach(), index, scaling, base.detach(), grad)
    _check(y.detach(), *want["y"])
    for name, g in zip(("dx", "ddown", "dup"), got):
        _check(g, *want[name])
    assert torch.equal(got[3], grad)
    again = torch.autograd.grad(y, leaves, grad, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for i, leaf in enumerate(leaves):                    # each gradient alone
        (one,) = torch.autograd.grad(y, (leaf,), grad, retain_graph=True)
        assert torch.equal(one, got[i])
    assert _lib.lib().bw_device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradients_against_differences(dtype):
    """y is linear in x, in down and in up: differences are exact but for the roundings of the two results (half a step of each) and of the gradient."""
    M, K, N, n, r = 37, 256, 192, 3, 16
    x, down, up, index, scaling, _ = _bank(M, K, N, n, r, dtype, seed=4)
    leaves = [t.requires_grad_() for t in (x, down, up)]
    grad = torch.randn(M, N, generator=_gen(5), device=DEV).to(dtype)
    got = torch.autograd.grad(adapter_matmul(*leaves, index, scaling=scaling), leaves, grad)
    half = torch.finfo(dtype).eps / 2
    with torch.no_grad():
        for i, g in enumerate(got):
            step = torch.randn(leaves[i].shape, generator=_gen(6 + i), device=DEV).sign().to(dtype) * leaves[i].abs().amax()
            ends = []
            for s in (1, -1):
                args = [t + s * step if j == i else t for j, t in enumerate(leaves)]
                moved = (args[i].double() - leaves[i].double()) if s == 1 else moved - (args[i].double() - leaves[i].double())
                ends.append(adapter_matmul(*args, index, scaling=scaling).double())
            want = (grad.double() * (ends[0] - ends[1])).sum()
            most = (grad.double().abs() * (ends[0].abs() + ends[1].abs())).sum() * (half + 2.0 ** -12) + (g.double() * moved).abs().sum() * (half + 2.0 ** -12)
            assert abs((g.double() * moved).sum() - want) <= most
            # the roundings are independent: a wrong formula is off by far more than this
            assert abs((g.double() * moved).sum() - want) <= 0.05 * (g.double() * moved).norm() + 0.05 * want.abs()


@pytest.mark.parametrize("K,N,r,M", [(512, 256, 16, 40), (100, 130, 5, 12), (512, 256, 16, 200)])
def test_rows_without_an_adapter_and_beyond_the_bank(K, N, r, M):
    """What stands in rows without an adapter reaches no other row and no sum; an index beyond the bank is loud."""
    x, down, up, index, scaling, base = _bank(M, K, N, 3, r, torch.float16, seed=7)
    index[5], index[6] = -1, -2 ** 31
    grad = torch.randn(M, N, generator=_gen(8), device=DEV).half()
    want = _formula(x, down, up, index, scaling, base, grad)
    x[index < 0], grad[index < 0] = math.nan, math.inf
    index[9] = 3
    leaves = [t.requires_grad_() for t in (x, down, up)]
    y = adapter_matmul(*leaves, index, scaling=scaling, base=base)
    dx, ddown, dup = torch.autograd.grad(y, leaves, grad)
    rest = torch.arange(M, device=DEV) != 9
    _check(y.detach()[rest], want["y"][0][rest], want["y"][1][rest])
    _check(dx[rest], want["dx"][0][rest], want["dx"][1][rest])
    assert bool(y[9].isnan().all()) and bool(dx[9].isnan().all()) and bool((dx[index < 0] == 0).all())
    # (row 9 had an adapter in the formula's sums or none; without it)
    index2 = index.clone()
    index2[9] = -1
    clean = [torch.where(index2[:, None] < 0, 0, t.detach()) for t in (x, grad)]
    again = _formula(clean[0], down.detach(), up.detach(), index2, scaling, base, clean[1])
    _check(ddown, *again["ddown"])
    _check(dup, *again["dup"])
    # a row of NaN that has an adapter reaches its own outputs and its adapter's sums alone
    t = int((index == 0).nonzero()[0, 0])
    x2 = x.detach().clone()
    x2[t] = math.nan
    y2 = adapter_matmul(x2, down.detach(), up.detach(), index, scaling=scaling, base=base)
    keep = torch.arange(M, device=DEV) != t
    assert bool(y2[t].isnan().all()) and torch.equal(y2[keep & rest], y.detach()[keep & rest])


@pytest.mark.parametrize("dtype,size", [(torch.float16, 1e-4), (torch.float16, 60.0), (torch.bfloat16, 1e-6), (torch.bfloat16, 1e9)])
def test_rank_values_far_from_one(dtype, size):
    """Gradients of fp16 models without loss scaling, and rank values beyond fp16's range, keep their precision."""
    M, K, N, n, r = 100, 512, 256, 2, 16
    x, down, up, index, scaling, _ = _bank(M, K, N, n, r, dtype, seed=9)
    x = (x * size).to(dtype)
    if dtype == torch.float16 and size > 1:
        down, up = (down * 400).to(dtype), (up * 2.0 ** -12).to(dtype)         # h of about 3e5
    leaves = [t.requires_grad_() for t in (x, down, up)]
    grad = (torch.randn(M, N, generator=_gen(10), device=DEV) * (size if size < 1 else 1.0)).to(dtype)
    y = adapter_matmul(*leaves, index, scaling=scaling)
    want = _formula(x.detach(), down.detach(), up.detach(), index, scaling, None, grad)
    _check(y.detach(), *want["y"])
    for name, g in zip(("dx", "ddown", "dup"), torch.autograd.grad(y, leaves, grad)):
        _check(g, *want[name])


def test_shapes_strides_and_empty_batches():
    x, down, up, index, scaling, base = _bank(24, 256, 320, 3, 16, torch.float16, seed=11)
    want = adapter_matmul(x, down, up, index, scaling=scaling, base=base)
    assert torch.equal(adapter_matmul(x.view(2, 3, 4, 256), down, up, index.view(2, 3, 4), scaling=scaling, base=base.view(2, 3, 4, 320)).view(24, 320), want)
    wide = torch.zeros(24, 300, dtype=torch.float16, device=DEV)
    wide[:, 3:259] = x
    assert torch.equal(adapter_matmul(wide[:, 3:259], down, up, index, scaling=scaling, base=base), want)
    cols = up.transpose(1, 2).contiguous()                                    # a checkpoint's lora_B
    assert torch.equal(adapter_matmul(x, down, cols.transpose(1, 2), index, scaling=scaling, base=base.T.contiguous().T), want)
    off = torch.zeros(24 * 256 + 1, dtype=torch.float16, device=DEV)
    off[1:] = x.flatten()
    got = adapter_matmul(off[1:].view(24, 256), down, up, index, scaling=scaling, base=base)      # rows off a 16-byte boundary
    _check(got, *_formula(x, down, up, index, scaling, base)["y"])
    leaves = [t[:0].requires_grad_() if t is x else t.requires_grad_() for t in (x, down, up)]
    y = adapter_matmul(*leaves, index[:0], scaling=scaling, base=base[:0])
    assert y.shape == (0, 320)
    dx, ddown, dup = torch.autograd.grad(y.sum(), leaves)
    assert dx.shape == (0, 256) and bool((ddown == 0).all()) and bool((dup == 0).all())


@pytest.mark.parametrize("M,n", [(70000, 2), (33000, 5), (40000, 1)])
def test_gradients_of_more_tokens_than_one_window(M, n):
    """Tokens are gathered from windows of 32768; an adapter may have none in the first, or all."""
    x, down, up, index, scaling, _ = _bank(M, 64, 72, n, 8, torch.float16, seed=12)
    if n == 2:
        index[:40000] = 0                   # the other one begins in the second window
    leaves = [t.requires_grad_() for t in (x, down, up)]
    grad = torch.randn(M, 72, generator=_gen(13), device=DEV).half()
    y = adapter_matmul(*leaves, index, scaling=scaling)
    want = _formula(x.detach(), down.detach(), up.detach(), index, scaling, None, grad)
    _check(y.detach(), *want["y"])
    for name, g in zip(("dx", "ddown", "dup"), torch.autograd.grad(y, leaves, grad)):
        _check(g, *want[name])


def test_graphs_of_forward_and_backward():
    """Captured training steps replayed beside each other and beside eager calls."""
    sets = []
    for i in range(2):
        x, down, up, index, scaling, base = _bank(130, 512, 256, 3, 16, torch.bfloat16, seed=20 + i)
        grad = torch.randn(130, 256, generator=_gen(30 + i), device=DEV).bfloat16()

        def step(x=x, down=down, up=up, index=index, scaling=scaling, base=base, grad=grad):
            leaves = [t.detach().requires_grad_() for t in (x, down, up)]
            y = adapter_matmul(*leaves, index, scaling=scaling, base=base)
            return [y.detach(), *torch.autograd.grad(y, leaves, grad)]

        sets.append(step)
    want = [step() for step in sets]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for step in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for out in outs:
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        eager = [step() for step in sets]
        torch.cuda.synchronize()
        for a, b, c in zip(outs, eager, want):
            assert all(torch.equal(p, q) and torch.equal(p, s) for p, q, s in zip(a, b, c))


def _packed(K, N, seed):
    lin = torch.nn.Linear(K, N, bias=True).to(DEV)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(N, K, generator=_gen(seed), device=DEV) * 0.02)
        lin.bias.copy_(torch.randn(N, generator=_gen(seed + 1), device=DEV) * 0.02)
    return QuantizedLinear.from_float(lin, bits=4, group_size=64)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_adapted_linear(dtype):
    layer = _packed(512, 768, 40)
    adapted = AdaptedLinear(layer, 3, 16, scaling=2.0, dtype=dtype)
    x = torch.randn(2, 21, 512, generator=_gen(42), device=DEV).to(dtype)
    index = torch.randint(-1, 3, (2, 21), generator=_gen(43), device=DEV).to(torch.int32)
    base = adapted(x, torch.full_like(index, -1))
    assert torch.equal(adapted(x, index), base)                         # new adapters change nothing
    with torch.no_grad():
        adapted.up.copy_(torch.randn(adapted.up.shape, generator=_gen(44), device=DEV) * 0.1)
        quiet = adapted(x, index)
    x.requires_grad_()
    y = adapted(x, index)
    assert torch.equal(y.detach(), quiet) and y.dtype == dtype
    args = (x.detach().view(42, 512), adapted.down.detach(), adapted.up.detach(), index.view(42), adapted.scaling)
    grad = torch.randn(2, 21, 768, generator=_gen(45), device=DEV).to(dtype)
    want = _formula(*args, base.detach().view(42, 768), grad.view(42, 768))
    _check(y.detach().view(42, 768), *want["y"])
    y.backward(grad)
    _check(adapted.down.grad, *want["ddown"])
    _check(adapted.up.grad, *want["dup"])
    # x has two gradients, each rounded, and their sum rounded
    x2 = x.detach().requires_grad_()
    adapted(x2, torch.full_like(index, -1)).backward(grad)
    both = x2.grad.double().view(42, 512) + want["dx"][0]
    half = torch.finfo(dtype).eps / 2
    most = half * (both.abs() + want["dx"][0].abs() + 1e-6) * 1.01 + 2.0 ** -12 * want["dx"][1] + 2.0 ** -24
    assert bool(((x.grad.double().view(42, 512) - both).abs() <= most).all())
    assert set(adapted.state_dict()) == {"down", "up", "scaling", "layer.qweight", "layer.scale", "layer.zero_point", "layer.bias"}


def test_an_attention_block_decodes_with_adapters_and_a_quantised_cache():
    """A run of them as a server makes it: packed projections with an adapter a request, the new rows appended, attention, the output
    projection; a prompt token by token gives what the same formulas give in 64 bits on the rows that the cache holds."""
    hidden, heads, kv_heads, dim, batch, steps = 512, 8, 2, 64, 3, 20
    wq, wk, wv, wo = (AdaptedLinear(_packed(hidden, n, 50 + i), 2, 8) for i, n in enumerate((heads * dim, kv_heads * dim, kv_heads * dim, hidden)))
    for i, w in enumerate((wq, wk, wv, wo)):
        with torch.no_grad():
            w.up.copy_(torch.randn(w.up.shape, generator=_gen(60 + i), device=DEV) * 0.1)
    index = torch.tensor([0, -1, 1], dtype=torch.int32, device=DEV)
    cache = QuantizedKVCache(9, 16, kv_heads, dim, bits=8, device=DEV)
    table = torch.tensor([[4, 1], [0, 7], [8, 3]], dtype=torch.int32, device=DEV)
    lengths = torch.zeros(batch, dtype=torch.int32, device=DEV)
    with torch.no_grad():
        for t in range(steps):
            x = torch.randn(batch, hidden, generator=_gen(70 + t), device=DEV).half()
            q, k, v = wq(x, index), wk(x, index), wv(x, index)
            cache.append(k.view(batch, kv_heads, dim), v.view(batch, kv_heads, dim), table[:, t // 16].long() * 16 + t % 16)
            lengths += 1
            a = cache.attend(q.view(batch, heads, dim), table, lengths)
            out = wo(a.view(batch, heads * dim), index)
    pos = torch.arange(steps, device=DEV)
    half = 2.0 ** -11
    for b in range(batch):
        k, v = (r.double().repeat_interleave(heads // kv_heads, 1) for r in cache.read(table[b, pos // 16].long() * 16 + pos % 16, dtype=torch.float32))
        w = torch.softmax(torch.einsum("hd,thd->ht", q[b].view(heads, dim).double(), k) * dim ** -0.5, -1)
        want, size = torch.einsum("ht,thd->hd", w, v), torch.einsum("ht,thd->hd", w, v.abs())
        assert bool(((a[b].double() - want).abs() <= half * want.abs() + half * size + 1e-6).all())
    assert torch.equal(out[1], wo.layer(a.view(batch, -1))[1]) and not torch.equal(out[0], wo.layer(a.view(batch, -1))[0])
    assert bool(out.isfinite().all())


@pytest.mark.parametrize("M, N, n, r, dtype", [
    (512, 264, 1, 64, torch.bfloat16), (513, 520, 1, 40, torch.float16), (1023, 2048, 2, 128, torch.bfloat16), (1500, 72, 2, 104, torch.float16),
    (2049, 136, 3, 24, torch.float16), (2048, 1000, 1, 32, torch.bfloat16), (17000, 128, 2, 64, torch.float16), (16385, 264, 1, 64, torch.bfloat16),
    (4096, 4096, 8, 64, torch.bfloat16), (4100, 14336, 4, 72, torch.float16)])
def test_gradients_of_many_tokens(M, N, n, r, dtype):
    """Sizes at which sums over tokens are formed on tcgen05: ragged stages, columns, rank blocks, lists and windows; tokens in no order."""
    x, down, up, index, scaling, base = _bank(M, 64, N, n, r, dtype, seed=60)
    grad = torch.randn(M, N, generator=_gen(61), device=DEV).to(dtype)
    leaves = [t.requires_grad_() for t in (x, down, up)]
    y = adapter_matmul(*leaves, index, scaling=scaling, base=base)
    dx, ddown, dup = torch.autograd.grad(y, leaves, grad)
    want = _formula(x.detach(), down.detach(), up.detach(), index, scaling, base, grad)
    for got, name in ((y.detach(), "y"), (dx, "dx"), (ddown, "ddown"), (dup, "dup")):
        _check(got, *want[name])
    assert _lib.lib().bw_device_status() == 0


@pytest.mark.parametrize("M, K, N, n, r, order, dtype", [
    (1027, 64, 8200, 1, 64, "any", torch.float16), (2050, 128, 12296, 3, 128, "any", torch.bfloat16), (6300, 64, 4000, 5, 40, "runs", torch.float16),
    (24600, 64, 1032, 2, 48, "any", torch.bfloat16), (3200, 256, 8064, 12, 104, "runs", torch.float16), (2050, 64, 1288, 9, 16, "any", torch.bfloat16),
    (5000, 64, 8, 3, 8, "runs", torch.bfloat16), (4096, 512, 2048, 200, 64, "any", torch.float16)])
def test_results_of_many_tokens(M, K, N, n, r, order, dtype):
    """With a base, without one and over it; an index beyond the bank gives NaN in its rows alone."""
    x, down, up, index, scaling, base = _bank(M, K, N, n, r, dtype, seed=70, order=order)
    want = _formula(x, down, up, index, scaling, base)["y"]
    y = adapter_matmul(x, down, up, index, scaling=scaling, base=base)
    _check(y, *want)
    over = base.clone()
    assert adapter_matmul(x, down, up, index, scaling=scaling, base=over, out=over) is over and torch.equal(over, y)
    _check(adapter_matmul(x, down, up, index, scaling=scaling), *_formula(x, down, up, index, scaling, None)["y"])
    beyond = index.clone()
    beyond[::7] = n + 3
    z = adapter_matmul(x, down, up, beyond, scaling=scaling, base=base)
    assert bool(z[::7].isnan().all())
    keep = torch.ones(M, dtype=torch.bool, device=DEV)
    keep[::7] = False
    assert torch.equal(z[keep], y[keep])
    assert _lib.lib().bw_device_status() == 0
