"""Calls of rotary positions, rotated appends, windowed attention and log probabilities that their documentation allows and programs seldom make."""
import copy
import math

import pytest
import torch

from bitween_b200 import QuantizedKVCache, RotaryPositions, token_log_probs
from bitween_b200.kernels import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_lib, "_operators", _lib._NoOperators)


def test_one_tensor_twice_and_shared_heads(path):
    r = RotaryPositions(64, 50)
    p = torch.arange(9, device=DEV)
    x = torch.randn(9, 2, 64, generator=_gen(1), device=DEV).half().requires_grad_()
    a, b = r.rotate(p, x, x)
    assert torch.equal(a, b)
    (twice,) = torch.autograd.grad((a, b), x, (torch.ones_like(a), torch.ones_like(a)))
    (once,) = torch.autograd.grad(r.rotate(p, x), x, torch.ones_like(a))
    assert torch.equal(twice, once * 2)
    shared = x.detach()[:, :1].expand(9, 5, 64).clone()[:, :1].requires_grad_()          # one head read as five
    y = r.rotate(p, shared.expand(9, 5, 64))
    assert all(torch.equal(y[:, h], y[:, 0]) for h in range(5)) and torch.equal(y[:, :1], r.rotate(p, shared))
    (g,) = torch.autograd.grad(y, shared, torch.ones_like(y))
    # five equal fp16 gradients added: exact in fp32, rounded once
    assert torch.equal(g, (once[:, :1].float() * 5).half())
    one = shared.detach()[:1].requires_grad_()                                           # one token's rows for all positions
    (g,) = torch.autograd.grad(r.rotate(p, one.expand(9, 1, 64)), one, torch.ones(9, 1, 64, device=DEV).half())
    assert bool(((g.double() - once[:, :1].double().sum(0, keepdim=True)).abs() <= 2.0 ** -11 * 20).all())


def test_empty_calls(path):
    r = RotaryPositions(64, 50, sections=(8, 12, 12))
    empty = torch.zeros(0, 2, 64, device=DEV).half().requires_grad_()
    at = torch.zeros(3, 0, dtype=torch.int64, device=DEV)
    y = r.rotate(at, empty)
    assert y.shape == (0, 2, 64)
    assert torch.autograd.grad(y, empty, torch.zeros_like(y))[0].shape == (0, 2, 64)
    x = torch.randn(4, 2, 64, generator=_gen(2), device=DEV).half()
    none, some = r.rotate(torch.zeros(4, dtype=torch.int64, device=DEV), x[:, :0], x)    # no heads
    assert none.shape == (4, 0, 64) and torch.equal(some, x)
    cache = QuantizedKVCache(0, 16, 2, 64, bits=4, device=DEV)                            # no pages: every slot is outside
    p = torch.arange(4, device=DEV)
    assert torch.equal(cache.append_rotated(x, x, x, p, r, p), r.rotate(p, x))
    table, lengths = torch.zeros(4, 3, dtype=torch.int32, device=DEV), torch.tensor([0, 5, 0, 48], dtype=torch.int32, device=DEV)
    out = cache.attend(x, table, lengths, window=4, sinks=1)
    assert not bool(out[[0, 2]].any()) and bool(out[[1, 3]].isnan().all())
    logits = torch.zeros(0, 70, device=DEV, requires_grad=True)
    got = token_log_probs(logits, torch.zeros(0, dtype=torch.int64, device=DEV), entropy=True, top=2)
    assert [tuple(t.shape) for t in got] == [(0,), (0,), (0, 2), (0, 2)]
    assert torch.autograd.grad(got.log_probs.sum() + got.entropy.sum(), logits)[0].shape == (0, 70)


def test_log_probs_of_parts(path):
    """What is not asked for is None, and gradients come from whatever was asked for."""
    x = torch.randn(5, 300, generator=_gen(3), device=DEV).requires_grad_()
    t = torch.tensor([3, 299, -1, 0, 7], device=DEV)
    assert token_log_probs(x) == (None, None, None, None)
    full = token_log_probs(x, t, entropy=True, top=4)
    for kw in ({"entropy": True}, {"top": 4}, {"entropy": True, "top": 4}):
        r = token_log_probs(x, **kw)
        assert r.log_probs is None
        for name in ("entropy", "top_log_probs", "top_tokens"):
            a, b = getattr(r, name), getattr(full, name)
            assert a is None or torch.equal(a, b)
        outs = [y for y in (r.entropy, r.top_log_probs) if y is not None]
        ws = [torch.randn(y.shape, generator=_gen(4), device=DEV) for y in outs]
        (a,) = torch.autograd.grad(outs, x, ws)
        (b,) = torch.autograd.grad([getattr(full, n) for n in ("entropy", "top_log_probs") if getattr(r, n) is not None], x, ws, retain_graph=True)
        assert torch.equal(a, b)
    assert not full.top_tokens.requires_grad and full.entropy.requires_grad
    wide = x.detach()[:1].requires_grad_()                                # one row, broadcast: its gradient is the rows' sum
    many = torch.arange(40, device=DEV) * 7
    (g,) = torch.autograd.grad(token_log_probs(wide.expand(40, 300), many).log_probs.sum(), wide)
    p = torch.softmax(wide.detach().double(), -1)
    want = torch.zeros(1, 300, dtype=torch.float64, device=DEV).index_add_(1, many, torch.ones(1, 40, dtype=torch.float64, device=DEV)) - 40 * p
    # 40 fp32 gradients of up to 1, each good to 2^-20, added in fp32
    assert bool(((g.double() - want).abs() <= 40 * 2.0 ** -20).all())


def test_a_copied_table_and_long_positions():
    r = RotaryPositions(32, 300000, base=500000.0, interleaved=True)
    p = torch.tensor([0, 1, 131071, 299999], device=DEV)
    x = torch.randn(4, 3, 32, generator=_gen(5), device=DEV)
    y = r.rotate(p, x)
    assert torch.equal(copy.deepcopy(r).rotate(p, x), y) and torch.equal(y[0], x[0])
    angle = p.double()[:, None] * 500000.0 ** (-torch.arange(16, device=DEV, dtype=torch.float64) / 16)
    z = torch.view_as_complex(x.double().unflatten(-1, (-1, 2)).contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None]
    # cosines of angles of up to 3e5 in 64 bits are good to 2^-34; rounded to fp32 2^-25, products and sums 2^-24 of |z| sqrt(2) each
    assert bool(((torch.view_as_real(z).flatten(-2) - y.double()).abs() <= 2.0 ** -21 * z.abs().repeat_interleave(2, -1)).all())


def test_rows_behind_the_last_are_left_as_they_were():
    """Pages and rows that no slot of a call names keep every bit, and so does the cache where all slots are padding."""
    r = RotaryPositions(128, 100)
    cache = QuantizedKVCache(6, 16, 2, 128, bits=8, device=DEV)
    for t in (cache.k_codes, cache.v_codes):
        t.random_(generator=_gen(6))
    cache.params.uniform_(-1, 1, generator=_gen(7))
    before = [t.clone() for t in cache._cache[:3]]
    x = torch.randn(40, 2, 128, generator=_gen(8), device=DEV).bfloat16()
    p = torch.arange(40, device=DEV)
    cache.append_rotated(x, x, x, torch.full((40,), -1, device=DEV), r, p)
    assert all(torch.equal(a, b) for a, b in zip(before, cache._cache[:3]))
    slots = torch.cat((torch.arange(17, 37, device=DEV), torch.tensor([96, -7, 2 ** 40, 1 << 33] * 5, device=DEV)))
    cache.append_rotated(x, x, x, slots, r, p)
    kept = torch.ones(96, dtype=torch.bool, device=DEV)
    kept[17:37] = False
    for a, b in zip(before, cache._cache[:3]):
        a, b = (t.transpose(1, 2).flatten(0, 1) for t in (a, b))
        assert torch.equal(a[kept], b[kept]) and not bool((a[~kept] == b[~kept]).all())


def test_log_probs_of_bf16_rows_at_the_edges():
    """The type's lowest value as a mask, rows of nothing else, and large offsets."""
    lowest = torch.finfo(torch.bfloat16).min
    for vocab in (17, 50272, 131071):
        x = (2 * torch.randn(6, vocab, generator=_gen(9), device=DEV)).bfloat16()
        x[0] = lowest
        x[1, 3:] = lowest
        x[2] += 3000
        x[3] = -math.inf
        x[3, 5] = lowest
        x[4, 1:] = -math.inf
        x[5] = -lowest
        t = torch.full((6,), 1, device=DEV)
        r = token_log_probs(x, t, entropy=True, top=min(3, vocab))
        lp = torch.log_softmax(x.double(), -1)
        h = torch.special.entr(lp.exp()).sum(-1)
        assert torch.equal(r.top_tokens, torch.sort(x.float(), descending=True, stable=True).indices[:, :3])
        for got, want in ((r.log_probs, lp[:, 1]), (r.entropy, h)):
            ok = want.isfinite()
            assert torch.equal(got.double()[~ok], want[~ok])
            # (a sum of equal terms, or of some units; results of up to 3e38 have their own rounding)
            assert bool(((got.double() - want)[ok].abs() <= 2.0 ** -16 + 2.0 ** -23 * want[ok].abs()).all()), vocab


def test_windows_on_threads_of_their_own_streams():
    import threading
    cache = QuantizedKVCache(400, 16, 2, 128, bits=4, device=DEV)
    rows = torch.randn(6400, 4, 128, generator=_gen(10), device=DEV).half()
    cache.append(rows[:, :2], rows[:, 2:], torch.arange(6400, device=DEV))
    q = torch.randn(20, 8, 128, generator=_gen(11), device=DEV).half()
    table = torch.randint(0, 400, (20, 400), generator=_gen(12), device=DEV, dtype=torch.int32)
    n = torch.randint(0, 6400, (20,), generator=_gen(13), device=DEV, dtype=torch.int32)
    kinds = [{"window": w, "sinks": s} for w, s in ((3000, 4), (17, 0), (0, 100), (6400, 6400))]
    want = [cache.attend(q, table, n, **kw) for kw in kinds]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(40):
                if not torch.equal(cache.attend(q, table, n, **kinds[i]), want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_and_overlapping_rows(dtype):
    """Rows of 30 million values, whose blocks are hundreds of steps; rows that begin inside each other."""
    x = (2 * torch.randn(2, 30000001, generator=_gen(14), device=DEV)).to(dtype)
    x[1, 29999990:] = 7.5
    t = torch.tensor([29999999, 0], device=DEV)
    r = token_log_probs(x, t, entropy=True, top=32)
    assert torch.equal(r.top_tokens, torch.sort(x.float(), descending=True, stable=True).indices[:, :32])
    lp = torch.log_softmax(x.double(), -1)
    h = torch.special.entr(lp.exp()).sum(-1)
    # spans of 25: 2^-22 of them for a weight's exponent, sums of some hundred parts a thread (2^-17 of a sum of parts of one sign)
    assert bool(((r.log_probs.double() - lp.gather(1, t[:, None])[:, 0]).abs() <= 2.0 ** -16).all())
    assert bool(((r.entropy.double() - h).abs() <= 2.0 ** -15 * 20).all())
    flat = x[0, :100000]
    rows = flat.as_strided((50, 5000), (1201, 1))
    a, b = token_log_probs(rows, top=3, entropy=True), token_log_probs(rows.contiguous(), top=3, entropy=True)
    assert torch.equal(a.top_tokens, b.top_tokens)
    # (pieces begin elsewhere in a row: the same sums in another order)
    assert bool(((a.entropy - b.entropy).abs() <= 2.0 ** -18 * 10).all())


def test_one_value_and_few():
    """Vocabularies of 1 to 40, each as dense rows and as rows off their boundaries: fewer values than threads, pieces or alternatives' groups."""
    for vocab in range(1, 41):
        big = torch.randn(9, vocab + 3, generator=_gen(vocab), device=DEV)
        for x in (big[:, :vocab].contiguous(), big[:, 1:1 + vocab], big[:, 2:2 + vocab].half(), big.bfloat16()[:, 3:3 + vocab]):
            t = torch.arange(9, device=DEV) % vocab
            top = min(vocab, 32)
            x = x.detach().requires_grad_()
            r = token_log_probs(x, t, entropy=True, top=top)
            lp = torch.log_softmax(x.detach().double(), -1)
            assert torch.equal(r.top_tokens, torch.sort(x.detach().float(), descending=True, stable=True).indices[:, :top])
            assert bool(((r.log_probs.double() - lp.gather(1, t[:, None])[:, 0]).abs() <= 2.0 ** -18).all())
            assert bool(((r.top_log_probs.double() - lp.gather(1, r.top_tokens)).abs() <= 2.0 ** -18).all())
            (g,) = torch.autograd.grad(r.log_probs, x, torch.ones(9, device=DEV))
            want = -lp.exp()
            want[torch.arange(9, device=DEV), t] += 1
            # (the token's entry is 1 - p from parts good to 2^-20)
            assert bool(((g.double() - want).abs() <= 2.0 ** -18 + torch.finfo(x.dtype).eps / 2 * want.abs()).all())


def test_numbers_of_other_types():
    np = pytest.importorskip("numpy")
    cache = QuantizedKVCache(4, 16, 2, 64, bits=4, device=DEV)
    x = torch.randn(3, 2, 64, generator=_gen(15), device=DEV).half()
    cache.append(x, x, torch.arange(3, device=DEV))
    table, n = torch.zeros(3, 1, dtype=torch.int32, device=DEV), torch.full((3,), 3, dtype=torch.int32, device=DEV)
    want = cache.attend(x, table, n, window=2, sinks=1)
    assert torch.equal(cache.attend(x, table, n, window=np.int64(2), sinks=np.int32(1)), want)
    assert torch.equal(cache.attend(x, table, n, window=2, sinks=True), want)
    logits = torch.randn(3, 50, generator=_gen(16), device=DEV)
    a, b = token_log_probs(logits, entropy=np.bool_(True), top=np.int64(4)), token_log_probs(logits, entropy=True, top=4)
    assert torch.equal(a.entropy, b.entropy) and torch.equal(a.top_tokens, b.top_tokens)
    with pytest.raises(TypeError):
        token_log_probs(logits, top=1.5)


@pytest.mark.parametrize("rows,vocab", [(160, 300), (160, 4000), (2100, 7000), (30, 500), (30, 8000), (200, 15000), (1300, 20000), (1300, 40), (2100, 2000)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_many_short_rows_with_masks(rows, vocab, dtype):
    """Rows that take CTAs of fewer threads, half of them masked (so that alternatives tie), some of one value, with gradients."""
    x = (2.5 * torch.randn(rows, vocab, generator=_gen(20), device=DEV)).to(dtype)
    x[::2, vocab // 7:] = -math.inf
    x[1::7] = 0.5
    x[2::9, vocab // 2:] = torch.finfo(dtype).min
    x[5] = -math.inf
    x[6, vocab // 3] = math.nan
    t = torch.randint(-1, max(1, vocab // 7), (rows,), generator=_gen(21), device=DEV)
    top = min(vocab, 32)
    x.requires_grad_()
    r = token_log_probs(x, t, entropy=True, top=top)
    d = x.detach().double()
    lp = torch.log_softmax(d, -1)
    assert torch.equal(r.top_tokens, torch.sort(x.detach().float(), descending=True, stable=True).indices[:, :top])
    want = torch.where(t < 0, 0.0, lp.gather(1, t.clamp(min=0)[:, None])[:, 0])
    h = torch.special.entr(lp.exp()).sum(-1)
    for got, ref, slack in ((r.log_probs, want, 2.0 ** -17), (r.entropy, h, 2.0 ** -16), (r.top_log_probs, lp.gather(1, r.top_tokens), 2.0 ** -17)):
        # (spans of 25: exponents good to 2^-20, sums to 2^-19; values of the type's lowest have their own rounding)
        ok = ref.isfinite()
        skip = (t < 0) & ~ok if ref.dim() == 1 and got is r.log_probs else torch.zeros_like(ok)
        assert torch.equal(got.double()[~ok & ~skip].nan_to_num(nan=7.0), ref[~ok & ~skip].nan_to_num(nan=7.0))
        assert bool(((got.double() - ref)[ok].abs() <= slack + 2.0 ** -23 * ref[ok].abs()).all())
    (g,) = torch.autograd.grad(r.log_probs, x, torch.ones(rows, device=DEV))
    fine = lp.exp().isfinite().all(-1) & (t >= 0)
    ref = -lp.exp()
    ref[torch.arange(rows, device=DEV), t.clamp(min=0)] += 1
    assert bool(((g.double() - ref)[fine].abs() <= 2.0 ** -17 + torch.finfo(dtype).eps / 2 * ref[fine].abs()).all()) and not bool(g[t < 0].any())


@pytest.mark.parametrize("rows,vocab", [(20, 700), (200, 700), (160, 8191), (300, 15001), (150, 20003), (3, 100003)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("apart", [0, 1])
def test_gradients_of_rows_of_every_kind(rows, vocab, dtype, apart):
    """The gradient's CTAs of each size and number, of rows that start where their gradient does and of rows that start elsewhere."""
    big = (2.5 * torch.randn(rows, vocab + 5 * apart, generator=_gen(30), device=DEV)).to(dtype)
    x = big[:, apart:vocab + apart].detach().requires_grad_()
    t = torch.randint(0, vocab, (rows,), generator=_gen(31), device=DEV)
    t[0], t[-1] = 0, vocab - 1
    r = token_log_probs(x, t, entropy=True, top=2)
    g, e, k = (torch.randn(*s, generator=_gen(32 + i), device=DEV) for i, s in enumerate(((rows,), (rows,), (rows, 2))))
    (got,) = torch.autograd.grad((r.log_probs, r.entropy, r.top_log_probs), x, (g, e, k))
    lp = torch.log_softmax(x.detach().double(), -1)
    p, h = lp.exp(), torch.special.entr(lp.exp()).sum(-1)
    all_g = (g.double() + k.double().sum(-1))[:, None]
    want = p * (-all_g - e.double()[:, None] * (lp + h[:, None]))
    want.scatter_add_(1, t[:, None], g.double()[:, None])
    want.scatter_add_(1, r.top_tokens, k.double())
    size = p * (all_g.abs() + g.double().abs()[:, None] + k.double().abs().sum(-1)[:, None] + e.double().abs()[:, None] * ((lp + h[:, None]).abs() + h[:, None]))
    # exponents of spans of 25 good to 2^-20, relative; entries of tokens are sums of up to four parts
    off = 2.0 ** -17 * size + 2.0 ** -21 * (g.abs() + k.abs().sum(-1)).double()[:, None]
    assert bool(((got.double() - want).abs() <= off + torch.finfo(dtype).eps / 2 * (want.abs() + off) + 2.0 ** -130).all())
