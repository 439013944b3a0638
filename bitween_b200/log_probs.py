"""Log probabilities of given tokens, with the entropy and the likeliest alternatives, and their gradient: what evaluation of a quantised model,
serving and fine-tuning of adapters ask of its logits.  Computed by the sm_100a kernels behind bw_token_log_probs and
bw_token_log_probs_grad."""
import operator
from collections import namedtuple

import torch
from torch.autograd.function import once_differentiable

from .kernels import _lib

_FLOAT_DTYPES = (torch.float32, torch.float16, torch.bfloat16)

TokenLogProbs = namedtuple("TokenLogProbs", "log_probs entropy top_log_probs top_tokens")


def _forward(logits, tokens, entropy, top, keep, lead):
    """(log_probs, entropy, top_log_probs, top_tokens, stats) of logits [rows, vocab], the first four of the leading shape `lead`; None for what is not asked."""
    rows, vocab = logits.shape
    dev = logits.device
    lp = None if tokens is None else torch.empty(lead, dtype=torch.float32, device=dev)
    h = torch.empty(lead, dtype=torch.float32, device=dev) if entropy else None
    top_lp = torch.empty((*lead, top), dtype=torch.float32, device=dev) if top else None
    top_t = torch.empty((*lead, top), dtype=torch.int64, device=dev) if top else None
    stats = torch.empty((rows, 4), dtype=torch.float32, device=dev) if keep else None
    L = _lib.lib()
    with _lib.on_device(dev):
        rc = L.bw_token_log_probs(logits.data_ptr(), _lib.dtype_code(logits.dtype), rows, vocab, logits.stride(0),
                                  *(None if t is None else t.data_ptr() for t in (tokens, lp, h)), top,
                                  *(None if t is None else t.data_ptr() for t in (top_lp, top_t, stats)), _lib.raw_stream(dev))
    _lib.check(rc)
    return lp, h, top_lp, top_t, stats


def _dense(t):
    return None if t is None else t.to(torch.float32).contiguous()


class TokenLogProbsFunction(torch.autograd.Function):
    """apply(logits, tokens, entropy, top): what `token_log_probs` says, of arguments that it may have checked or not (a traced call runs again with other tensors)."""

    @staticmethod
    def forward(ctx, logits, tokens, entropy, top):
        x, tokens = _arguments(logits, tokens, top)
        lp, h, top_lp, top_t, stats = _forward(x, tokens, entropy, top, ctx.needs_input_grad[0], logits.shape[:-1])
        ctx.save_for_backward(x, tokens, top_t, stats)
        ctx.like = [None if t is None else (t.shape, t.dtype, t.device) for t in (x, tokens, top_t, stats)]
        ctx.top, ctx.shape = top, logits.shape
        ctx.set_materialize_grads(False)
        if top_t is not None:
            ctx.mark_non_differentiable(top_t)
        return lp, h, top_lp, top_t

    @staticmethod
    @once_differentiable
    def backward(ctx, g, e, g_top, _):
        _lib.refuse_capture("token_log_probs")
        saved = ctx.saved_tensors
        # (hooks may have made other tensors of them in the meantime: moved, packed)
        if any((t is None) != (like is None) or (t is not None and (t.shape, t.dtype, t.device) != like) for t, like in zip(saved, ctx.like)):
            raise RuntimeError("token_log_probs: a tensor saved for the backward pass has come back from its hooks in another shape, type or place")
        if not ctx.needs_input_grad[0] or (g is None and e is None and g_top is None):
            return None, None, None, None
        logits, tokens, top_t, stats = saved
        logits = _rows(logits)
        tokens, top_t, stats = (t if t is None else t.contiguous() for t in (tokens, top_t, stats))
        g, e, g_top = _dense(g), _dense(e), _dense(g_top)
        rows, vocab = logits.shape
        dev = logits.device
        grad = torch.empty(ctx.shape, dtype=logits.dtype, device=dev)
        L = _lib.lib()
        with _lib.on_device(dev):
            rc = L.bw_token_log_probs_grad(logits.data_ptr(), _lib.dtype_code(logits.dtype), rows, vocab, logits.stride(0),
                                           None if tokens is None else tokens.data_ptr(), stats.data_ptr(), *(None if t is None else t.data_ptr() for t in (g, e)), ctx.top,
                                           *(None if t is None else t.data_ptr() for t in (top_t, g_top)), grad.data_ptr(), _lib.raw_stream(dev))
        _lib.check(rc)
        return grad, None, None, None


def _rows(logits):
    logits = logits.resolve_neg()
    return logits if logits.stride(1) == 1 and logits.stride(0) >= 0 else logits.contiguous()


def _arguments(logits, tokens, top):
    """(logits [rows, vocab], tokens [rows]) of a call, checked, as the kernels take them."""
    _lib.require_cuda(logits, "logits")
    if logits.dtype not in _FLOAT_DTYPES:
        raise TypeError(f"token_log_probs: unsupported dtype {logits.dtype} (float32/float16/bfloat16)")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must be [..., vocab] of at least one token")
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    if not 0 <= top <= min(32, vocab):
        raise ValueError(f"top must be 0 to {min(32, vocab)}")
    if tokens is not None:
        if tokens.dtype != torch.int64:
            raise TypeError("tokens must be int64")
        if tokens.shape != lead:
            raise ValueError(f"tokens must have shape {tuple(lead)}")
        if tokens.device != logits.device:
            raise RuntimeError(f"`tokens` is on {tokens.device} but logits is on {logits.device}")
        tokens = tokens.reshape(-1).contiguous()
    return _rows(logits.reshape(-1, vocab)), tokens


def token_log_probs(logits, tokens=None, entropy=False, top=0):
    """log softmax of `logits` [..., vocab] (fp32, fp16 or bf16; rows may be strided) at `tokens` (int64, of the leading shape), as a tuple
    (log_probs, entropy, top_log_probs, top_tokens) with None for what is not asked:

    log_probs, entropy   fp32, of the leading shape.  A token below 0 has log probability 0 and no gradient (padding); one beyond the vocabulary gives NaN.
    top_log_probs, top_tokens   fp32 and int64 [..., top] (up to 32): the largest logits in falling order, equal ones by rising index.

    Where a probability is 0 (a logit of -infinity) it adds nothing to the entropy.  A row with NaN or +infinity, or of -infinity alone, gives NaN.
    Differentiable in the logits through log_probs, entropy and top_log_probs; the gradient is formed in fp32 and rounded once."""
    ops = _lib._operators or _lib.host_operators()
    out = ops.token_log_probs(logits, tokens, entropy, top)
    if out is not None:
        return TokenLogProbs._make(out)
    _lib.refuse_recorders("token_log_probs")
    entropy, top = bool(entropy), operator.index(top)
    x, t = (logits, tokens) if torch.jit.is_tracing() else _arguments(logits, tokens, top)
    if tokens is None and not entropy and not top:
        return TokenLogProbs(None, None, None, None)
    out = ops.token_log_probs(x, t, entropy, top)
    if out is not None:
        return TokenLogProbs(*(y if y is None else y.view((*logits.shape[:-1], *y.shape[1:])) for y in out))
    if not _lib.for_autograd(logits):
        return TokenLogProbs._make(_forward(x, t, entropy, top, False, logits.shape[:-1])[:4])
    del x, t                                             # (a copy of strided rows is made again)
    return TokenLogProbs._make(TokenLogProbsFunction.apply(logits, tokens, entropy, top))
