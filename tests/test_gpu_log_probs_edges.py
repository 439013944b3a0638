"""Log probabilities: what their documentation promises of tokens beyond the vocabulary, and of calls that differ in what is asked for."""
import pytest
import torch

from bitween_b200 import token_log_probs
from bitween_b200.kernels import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_lib, "_operators", _lib._NoOperators)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [50, 1003, 50272])
def test_a_token_beyond_the_vocabulary_that_nothing_is_asked_of(vocab, dtype, path):
    """A row whose gradients are all 0 gets zeros, as a loss that drops such tokens expects; one with a gradient of the token gets NaN; one with others' alone gets theirs."""
    x = (2.5 * torch.randn(7, vocab, generator=_gen(1), device=DEV)).to(dtype).requires_grad_()
    t = torch.tensor([vocab, 3, 2 ** 40, vocab, vocab, -1, vocab + 5], device=DEV)
    r = token_log_probs(x, t, entropy=True, top=3)
    assert r.log_probs.isnan().tolist() == [True, False, True, True, True, False, True]
    (dx,) = torch.autograd.grad(torch.where(t < vocab, r.log_probs, 0.0).sum(), x, retain_graph=True)
    assert not bool(dx[[0, 2, 3, 4, 5, 6]].any()) and bool(dx[1].any()) and bool(dx.isfinite().all())
    g, e, k = torch.tensor([0.0, 1, 0, 0, 2, 1, -0.0], device=DEV), torch.tensor([0.0, 0, 0, 3, 0, 0, 0], device=DEV), torch.zeros(7, 3, device=DEV)
    k[2, 1] = 1.5
    (dx,) = torch.autograd.grad((r.log_probs, r.entropy, r.top_log_probs), x, (g, e, k), retain_graph=True)
    assert not bool(dx[[0, 5, 6]].any()) and bool(dx[4].isnan().all()) and bool(dx[[1, 2, 3]].isfinite().all())
    # (the rows with other gradients are those of a call that has no tokens, bit for bit)
    bare = token_log_probs(x, entropy=True, top=3)
    (want,) = torch.autograd.grad((bare.entropy, bare.top_log_probs), x, (e, k))
    assert torch.equal(dx[[2, 3]], want[[2, 3]]) and bool(dx[[2, 3]].any(-1).all())


@pytest.mark.parametrize("rows,vocab", [(61, 50272), (200, 15000), (1300, 20000), (1300, 70001), (2100, 32000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_log_probs_whatever_else_is_asked_for(rows, vocab, dtype):
    """With and without the entropy bit for bit; with alternatives, for which other CTAs may take the row, to what the order of its sums leaves open."""
    x = (2.5 * torch.randn(rows, vocab, generator=_gen(2), device=DEV)).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=_gen(3), device=DEV)
    bare, with_h, some, all_of_it = (token_log_probs(x, t, entropy=e, top=k) for e, k in ((False, 0), (True, 0), (False, 5), (True, 5)))
    assert torch.equal(bare.log_probs, with_h.log_probs) and torch.equal(some.log_probs, all_of_it.log_probs)
    assert torch.equal(some.top_log_probs, all_of_it.top_log_probs) and torch.equal(some.top_tokens, all_of_it.top_tokens)
    # weights' exponents good to 2^-22 of spans of less than 32, relative, and sums of some hundred fp32 parts each to 2^-19; an entropy of less than 16 by twice that and its own 2^-24
    # each; on both sides
    assert bool(((bare.log_probs.double() - some.log_probs.double()).abs() <= 2 * (2.0 ** -17 + 2.0 ** -19)).all())
    assert bool(((with_h.entropy.double() - all_of_it.entropy.double()).abs() <= 4 * (2.0 ** -17 + 2.0 ** -19)).all())
