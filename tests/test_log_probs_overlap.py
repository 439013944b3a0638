"""A gradient of log probabilities that would be written over its own logits is refused."""
import pytest
import torch

from bitween_b200 import token_log_probs
from bitween_b200.kernels import _lib

P = 1 << 30      # an aligned address that no call here reaches


def test_gradients_over_the_logits_are_refused():
    L = _lib.lib()

    def grad(to, rows=3, vocab=100, stride=128, dtype=1):
        return L.bw_token_log_probs_grad(P, dtype, rows, vocab, stride, None, 16, None, 16, 0, None, None, to, None)

    # (fp16: rows of 200 bytes, 256 apart; a gradient of 600 bytes)
    for at in (0, 2, 198, -2, -598, 256, 456, 2 * 256 + 198, 254, 200):
        assert grad(P + at) == 9
    # rows behind each other, one row many times, one row
    assert grad(P, stride=100) == 9 and grad(P + 598, stride=100) == 9 and grad(P - 598, stride=100) == 9
    assert grad(P + 198, stride=0) == 9 and grad(P - 598, stride=0) == 9
    assert grad(P + 198, rows=1) == 9 and grad(P - 198, rows=1) == 9
    # rows that lie before the first one
    assert grad(P - 512, stride=-128) == 9 and grad(P - 512 - 598, stride=-128) == 9 and grad(P + 198, stride=-128) == 9


@pytest.mark.gpu
def test_gradients_between_and_beside_the_logits():
    """Dense gradients that lie in the gap between two rows, or right before or behind all of them."""
    L = _lib.lib()
    buffer = torch.randn(6000, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    tokens, g = torch.tensor([7, 63], device="cuda"), torch.tensor([1.0, -2.0], device="cuda")
    x = buffer[1000:].as_strided((2, 64), (2048, 1)).clone().requires_grad_()
    (want,) = torch.autograd.grad(token_log_probs(x, tokens).log_probs, x, g)
    stats, lp, stream = torch.empty(2, 4, device="cuda"), torch.empty(2, device="cuda"), torch.cuda.current_stream().cuda_stream
    logits = buffer[1000:].data_ptr()
    assert L.bw_token_log_probs(logits, 0, 2, 64, 2048, tokens.data_ptr(), lp.data_ptr(), None, 0, None, None, stats.data_ptr(), stream) == 0
    for at in (1000 - 128, 1064, 1000 + 2048 - 128, 1064 + 2048):
        before = buffer.clone()
        assert L.bw_token_log_probs_grad(logits, 0, 2, 64, 2048, tokens.data_ptr(), stats.data_ptr(), g.data_ptr(), None, 0, None, None, buffer[at:].data_ptr(), stream) == 0
        assert torch.equal(buffer[at:at + 128].view(2, 64), want)
        before[at:at + 128] = buffer[at:at + 128]
        assert torch.equal(before, buffer)
    assert L.bw_token_log_probs_grad(logits, 0, 2, 64, 2048, tokens.data_ptr(), stats.data_ptr(), g.data_ptr(), None, 0, None, None, buffer[1063:].data_ptr(), stream) == 9
    assert L.bw_device_status() == 0
