"""Log probabilities of tokens with entropy and alternatives, and their gradients, against 64-bit sums."""
import math

import pytest
import torch

from bitween_b200 import token_log_probs
from bitween_b200.kernels import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _logits(rows, vocab, dtype, seed, scale=2.5):
    return (scale * torch.randn(rows, vocab, generator=_gen(seed), device=DEV)).to(dtype)


def _want(x, tokens):
    """(log probabilities of all tokens, of the given ones, entropy) in 64 bits."""
    lp = torch.log_softmax(x.double(), -1)
    at = lp.gather(-1, tokens.clamp(0, x.shape[-1] - 1)[..., None])[..., 0]
    at = torch.where(tokens < 0, 0.0, torch.where(tokens >= x.shape[-1], math.nan, at))
    p = lp.exp()
    return lp, at, -torch.where(p == 0, 0.0, p * lp).sum(-1)


def _order(x, top):
    """Falling values, equal ones by rising index; NaN first (which torch's stable sort does)."""
    return torch.sort(x.float() + 0.0, dim=-1, descending=True, stable=True).indices[..., :top]


def _near(got, want, slack):
    assert got.dtype == torch.float32 and got.shape == want.shape
    bad = want.isnan() | want.isinf()
    assert torch.equal(got.double()[bad].nan_to_num(nan=7.0), want[bad].nan_to_num(nan=7.0))
    assert bool(((got.double() - want).abs()[~bad] <= slack.expand(want.shape)[~bad]).all())


def _slack(x):
    """Of a log probability: x - m and its product with 1/ln 2 have 2^-24 of |x - m| each, which shift a weight by as much; ln of a sum of fp32 parts (some hundred to a thread, then a
    tree) has 2^-19; the result's own rounding.  Of a span of values up to 2^5 together less than 2^-17."""
    span = torch.where(x.isfinite(), x.double(), 0.0)
    return 2.0 ** -22 * (span.amax(-1) - span.amin(-1) + 8)


SIZES = [(1, 1), (1, 2), (3, 7), (1, 50272), (61, 1000), (5, 4097), (300, 129), (2, 131071), (7, 32768), (600, 2053), (3, 262147)]


@pytest.mark.parametrize("rows,vocab", SIZES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_log_probs_entropy_and_alternatives(rows, vocab, dtype):
    x = _logits(rows, vocab, dtype, 1)
    tokens = torch.randint(0, vocab, (rows,), generator=_gen(2), device=DEV)
    tokens[rows // 2] = -100 if rows > 1 else tokens[0]
    lp, at, h = _want(x, tokens)
    slack = _slack(x)
    for top in sorted({0, 1, min(5, vocab), min(20, vocab), min(32, vocab)}):
        r = token_log_probs(x, tokens, entropy=True, top=top)
        _near(r.log_probs, at, slack)
        _near(r.entropy, h, 2 * slack)
        if top:
            order = _order(x, top)
            assert r.top_tokens.dtype == torch.int64 and torch.equal(r.top_tokens, order)
            _near(r.top_log_probs, lp.gather(-1, order), slack[:, None])
        else:
            assert r.top_tokens is None and r.top_log_probs is None
    bare = token_log_probs(x, tokens)
    assert bare.entropy is None and torch.equal(bare.log_probs, r.log_probs)
    none = token_log_probs(x, entropy=True)
    assert none.log_probs is None and torch.equal(none.entropy, r.entropy)
    assert _lib.lib().bw_device_status() == 0


@pytest.mark.parametrize("vocab", [1, 5, 40, 333, 5000, 50272, 131071, 300007])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_at_the_edges(vocab, dtype):
    """Equal values, masks, infinities, NaN: which alternatives come, and what is not a number."""
    x = _logits(17, vocab, dtype, 3)
    x[0] = 0.0
    x[1] = -math.inf
    x[2] = -math.inf
    x[2, vocab // 2] = 3.0
    x[3] = torch.finfo(dtype).min
    x[4, vocab // 3:] = torch.finfo(dtype).min
    x[5, vocab - 1] = math.inf
    x[6, vocab // 2] = math.nan
    x[7] = math.nan
    x[8, ::2] = 0.0
    x[8, 1::2] = -0.0
    x[9] = torch.arange(vocab, device=DEV) % 3                                       # many equal maxima
    x[10] = torch.linspace(-30, 30, vocab, device=DEV)                               # rising
    x[11] = torch.linspace(30, -30, vocab, device=DEV)                               # falling
    x[12] = -math.inf
    x[12, max(0, vocab - 3):] = 1.0
    x[13] *= 1000 if dtype == torch.float32 else 100
    x[14] = (torch.arange(vocab, device=DEV) % 4096 >= 4090).float() * 5             # maxima in few threads' places
    x[15] = torch.where(torch.arange(vocab, device=DEV) % 256 < 2, torch.arange(vocab, device=DEV) / vocab * 9, -4.0)
    x[16, :] = -5.0
    x[16, vocab // 4:vocab // 4 + 300] = 2.0
    tokens = torch.randint(0, vocab, (17,), generator=_gen(4), device=DEV)
    tokens[0] = vocab
    tokens[9] = 2 ** 40
    tokens[2] = vocab // 2
    top = min(20, vocab)
    r = token_log_probs(x, tokens, entropy=True, top=top)
    lp, at, h = _want(x, tokens)
    order = _order(x, top)
    assert torch.equal(r.top_tokens, order)
    slack = _slack(x)
    slack[13] *= 4
    _near(r.log_probs, at, slack)
    # (of spans of 10^3 and more a weight that is off by its exponent's rounding has been lost long before)
    _near(r.entropy, h, 2 * slack.clamp(max=2.0 ** -14))
    _near(r.top_log_probs, lp.gather(-1, order), slack[:, None])
    assert bool(r.entropy[[1, 5, 6, 7]].isnan().all())
    assert float(r.log_probs[2]) == 0.0 and float(r.entropy[2]) == 0.0


@pytest.mark.parametrize("vocab", [40, 9001, 131072])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_a_nan_beside_masked_values_is_not_lost(vocab, dtype):
    """NaN where nothing else of a thread's first values is finite, at every place in turn of some rows."""
    places = sorted({0, 1, 7, 8, 9, vocab // 3, vocab - 9, vocab - 1})
    x = torch.full((2 * len(places), vocab), -math.inf, device=DEV)
    x[:, vocab // 2:] = torch.randn(len(x), vocab - vocab // 2, generator=_gen(18), device=DEV)
    for i, at in enumerate(places):
        x[2 * i, at] = math.nan
        x[2 * i + 1, at] = math.inf
    x = x.to(dtype)
    r = token_log_probs(x, torch.full((len(x),), vocab - 2, device=DEV), entropy=True, top=3)
    assert bool(r.log_probs.isnan().all()) and bool(r.entropy.isnan().all()) and bool(r.top_log_probs.isnan().all())
    assert torch.equal(r.top_tokens, _order(x, 3))


def test_padding_reads_nothing_of_its_row():
    """Rows that no token, entropy or alternative is asked of: 0 and a gradient of 0, whatever stands in them."""
    x = _logits(6, 50272, torch.bfloat16, 19)
    x[1], x[4, 77] = math.nan, math.inf
    tokens = torch.tensor([5, -100, 9, 50271, -1, 0], device=DEV)
    x.requires_grad_()
    r = token_log_probs(x, tokens)
    (dx,) = torch.autograd.grad(r.log_probs, x, torch.ones(6, device=DEV))
    assert not bool(r.log_probs[[1, 4]].any()) and not bool(dx[[1, 4]].any()) and bool(dx[[0, 2, 3, 5]].isfinite().all()) and bool(dx[[0, 2, 3, 5]].any(-1).all())


def _grads(x, tokens, g, e, top_tokens=None, g_top=None):
    """The formula, and a bound of what fp32 leaves out: (gradient, size)."""
    lp, _, h = _want(x, tokens)
    p = lp.exp()
    g = torch.where(tokens < 0, 0.0, g.double())
    all_g = g + (0 if g_top is None else g_top.double().sum(-1))
    inner = torch.where(p == 0, 0.0, lp + h[:, None])
    out = p * (-all_g[:, None] - e.double()[:, None] * inner)
    out.scatter_add_(1, tokens.clamp(min=0)[:, None], g[:, None])
    if g_top is not None:
        out.scatter_add_(1, top_tokens, g_top.double())
    size = p * (all_g.abs()[:, None] + (0 if g_top is None else g_top.double().abs().sum(-1)[:, None]) + e.double().abs()[:, None] * (inner.abs() + h[:, None]))
    return out, size


@pytest.mark.parametrize("rows,vocab", [(1, 2), (3, 7), (1, 50272), (61, 1000), (5, 4097), (300, 129), (2, 131071), (64, 32768), (600, 2053)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_gradients(rows, vocab, dtype):
    x = _logits(rows, vocab, dtype, 5).requires_grad_()
    tokens = torch.randint(0, vocab, (rows,), generator=_gen(6), device=DEV)
    if rows > 2:
        tokens[rows // 2] = -100
    top = min(20, vocab)
    g, e = torch.randn(rows, generator=_gen(7), device=DEV), torch.randn(rows, generator=_gen(8), device=DEV)
    g_top = torch.randn(rows, top, generator=_gen(9), device=DEV)
    r = token_log_probs(x, tokens, entropy=True, top=top)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(r, token_log_probs(x, tokens, entropy=True, top=top)))
    half, zero = torch.finfo(dtype).eps / 2, torch.zeros_like(g)
    slack = _slack(x.detach())[:, None] * 2                              # of a probability, relative: its exponent's error; of inner by as much
    tiny = torch.finfo(dtype).smallest_normal * half
    for outs, gs, args in (((r.log_probs,), (g,), (g, zero)), ((r.entropy,), (e,), (zero, e)), ((r.log_probs, r.entropy), (g, e), (g, e)),
                           ((r.log_probs, r.top_log_probs, r.entropy), (g, g_top, e), (g, e, r.top_tokens, g_top)), ((r.top_log_probs,), (g_top,), (zero, zero, r.top_tokens, g_top))):
        (dx,) = torch.autograd.grad(outs, x, gs, retain_graph=True)
        want, size = _grads(x.detach(), tokens, *args)
        assert dx.dtype == dtype and dx.shape == x.shape
        # (the entries of the tokens are sums of two: 2^-23 of both)
        off = slack * size + 2.0 ** -22 * (want.abs() + size)
        assert bool(((dx.double() - want).abs() <= off + half * (want.abs() + off) + 2 * tiny).all())


def test_gradients_against_differences():
    x = _logits(5, 60, torch.float32, 10).requires_grad_()
    tokens = torch.tensor([3, -100, 59, 0, 31], device=DEV)
    w = torch.randn(3, 5, generator=_gen(11), device=DEV).double()
    w_top = torch.randn(5, 4, generator=_gen(12), device=DEV).double()

    def loss(y, order):
        lp, at, h = _want(y, tokens)
        return (w[0] * at + w[1] * h).sum() + (w_top * lp.gather(-1, order)).sum()

    r = token_log_probs(x, tokens, entropy=True, top=4)
    (dx,) = torch.autograd.grad((r.log_probs, r.entropy, r.top_log_probs), x, (w[0].float(), w[1].float(), w_top.float()))
    step, base = 1e-5, x.detach().double()
    for i in range(5):
        for j in range(0, 60, 7):
            d = torch.zeros_like(base)
            d[i, j] = step
            diff = (loss(base + d, r.top_tokens) - loss(base - d, r.top_tokens)) / (2 * step)
            # a central difference in 64 bits: step^2 of the third derivative (less than 100), and 2^-52 * 100 / step; fp32 gradients of some units: 2^-20
            assert abs(float(diff) - float(dx[i, j])) <= 1e-8 + 1e-8 + 2.0 ** -17


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_gradients_at_the_edges(dtype):
    vocab = 1003
    x = _logits(8, vocab, dtype, 13)
    x[0, 5:] = -math.inf
    x[1] = -math.inf
    x[2, 100] = math.inf
    x[3, 100] = math.nan
    x[4, 10:] = torch.finfo(dtype).min
    tokens = torch.tensor([2, 5, 100, 7, 3, vocab, -1, 9], device=DEV)
    x.requires_grad_()
    r = token_log_probs(x, tokens, entropy=True, top=3)
    g = torch.ones(8, device=DEV)
    (dx,) = torch.autograd.grad((r.log_probs, r.entropy), x, (g, g))
    nan = dx.isnan().any(-1)
    assert nan.tolist() == [False, True, True, True, False, True, False, False]
    assert bool(dx[[1, 2, 3, 5]].isnan().all())
    assert not bool(dx[0, 5:].any()) and not bool(dx[4, 10:].any())
    want, size = _grads(x.detach(), tokens.clamp(max=vocab - 1), g, g)
    ok = [0, 4, 6, 7]
    half = torch.finfo(dtype).eps / 2
    assert bool(((dx.double() - want)[ok].abs() <= half * want[ok].abs() + 2.0 ** -15 * size[ok] + 2.0 ** -24).all())
    # a token whose probability is 0 takes its gradient; the same token given and among the alternatives takes both
    (dx,) = torch.autograd.grad(token_log_probs(x, tokens.clone().fill_(8), top=3).log_probs, x, g)
    assert float(dx[0, 8]) == 1.0


def test_shapes_strides_and_offsets():
    big = _logits(12, 5003, torch.bfloat16, 14)
    x = big[:, 3:4099].unflatten(0, (3, 4))                               # rows that start anywhere
    tokens = torch.randint(0, 4096, (3, 4), generator=_gen(15), device=DEV)
    r = token_log_probs(x, tokens, entropy=True, top=7)
    dense = token_log_probs(x.contiguous(), tokens, entropy=True, top=7)
    lp, at, h = _want(x, tokens)
    assert r.log_probs.shape == (3, 4) and r.top_tokens.shape == (3, 4, 7)
    for got in (r, dense):
        _near(got.log_probs, at, _slack(x))
        _near(got.entropy, h, 2 * _slack(x))
        assert torch.equal(got.top_tokens, _order(x, 7))
    leaf = big.clone().requires_grad_()
    y = leaf[:, 3:4099].unflatten(0, (3, 4))
    token_log_probs(y, tokens).log_probs.sum().backward()
    want, size = _grads(x.flatten(0, 1), tokens.flatten(), torch.ones(12, device=DEV), torch.zeros(12, device=DEV))
    got = leaf.grad[:, 3:4099]
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -15 * size + 2.0 ** -130).all()) and not bool(leaf.grad[:, :3].any()) and not bool(leaf.grad[:, 4099:].any())
    one = token_log_probs(x[0, 0], tokens[0, 0], top=2)                   # no leading dimension
    assert one.log_probs.shape == () and one.top_tokens.shape == (2,) and float(one.log_probs) == float(r.log_probs[0, 0])
    assert token_log_probs(x[:0], tokens[:0], entropy=True, top=2).top_tokens.shape == (0, 4, 2)
    columns = x[0].T.contiguous().T
    assert torch.equal(token_log_probs(columns, tokens[0], top=7).top_tokens, r.top_tokens[0])
    rows = x[0, :1].expand(9, -1)                                         # one row many times
    assert torch.equal(token_log_probs(rows, tokens[0, :1].expand(9), top=7).top_tokens, r.top_tokens[0, :1].expand(9, -1))


def test_rows_past_32_bits():
    """Logits and a gradient of more than 2^31 values."""
    rows, vocab = 21000, 104729
    x = torch.empty((rows, vocab), dtype=torch.float16, device=DEV)
    for part in x.split(1000):
        part.copy_(2.5 * torch.randn(part.shape, generator=_gen(16), device=DEV))
    x.requires_grad_()
    tokens = torch.randint(0, vocab, (rows,), generator=_gen(17), device=DEV)
    r = token_log_probs(x, tokens, entropy=True, top=3)
    at = torch.tensor([0, 11111, 20480, 20999], device=DEV)
    some = x.detach()[at]
    lp, want, h = _want(some, tokens[at])
    _near(r.log_probs[at].detach(), want, _slack(some))
    assert torch.equal(r.top_tokens[at], _order(some, 3))
    (dx,) = torch.autograd.grad(r.log_probs, x, torch.ones(rows, device=DEV))
    want, size = _grads(some, tokens[at], torch.ones(4, device=DEV), torch.zeros(4, device=DEV))
    assert bool(((dx[at].double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -15 * size + 2.0 ** -24).all())


def test_graphs_and_streams():
    xs = [_logits(6, 50272, torch.bfloat16, 20 + i) for i in range(3)]
    tokens = torch.randint(0, 50272, (6,), generator=_gen(23), device=DEV)
    want = [token_log_probs(x, tokens, entropy=True, top=5) for x in xs]
    graphs, outs = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([token_log_probs(x, tokens, entropy=True, top=5) for _ in range(4)])
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        eager = [token_log_probs(x, tokens, entropy=True, top=5) for x in xs]
        torch.cuda.synchronize()
        for out, got, ref in zip(outs, eager, want):
            for r in (*out, got):
                assert all(torch.equal(a, b) for a, b in zip(r, ref))
