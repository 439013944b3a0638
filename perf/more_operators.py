"""What a decoding or fine-tuning step does around the packed linears and the cache, as cases that can be timed: rotary positions of one or
several axes, rows appended to the quantised cache with that rotation on the way, attention over the cache with a sliding window and
sinks, and the log probabilities of tokens with their gradient.

Where `own` is false, `run` computes them in elementary torch operations in 32 bits; where it is true, it makes the calls of this
package.  The formulas:

  rotate     pair j of a head's first R values is (j, j + R / 2), or (2 j, 2 j + 1) where interleaved.  With (c, s) the cosine and sine of position * R-th
             frequency j, rounded to fp32, the pair (a, b) becomes (a c - b s, b c + a s), each operation rounded in fp32.  The position is that of the pair's
             axis (time, height, width).  Values behind the first R stay.  Gradients are turned back: (a c + b s, b c - a s).
  append     the rotated queries; and rotated keys (in fp32), and values, quantised into the cache.  A row is one token's D values of one head.  With
             Q = 2^bits - 1, lo = min(row, 0), hi = max(row, 0): scale = (hi - lo) / Q rounded up to fp16, at least 2^-24;
             zero = round(-lo / scale); code = clamp(round(x / scale + zero), 0, Q).  A row stands for scale * (code - zero).
  attend     out[b, h] = sum_t softmax_t(q[b, h] . K[t, h / group] / sqrt(D)) V[t, h / group] over the t < lengths[b] of a paged cache that are among the
             first `sinks` or the last `window`.  Pages that hold none of those have been given up: the table has -1 there.
  log probs  of row x and token t: x[t] - log sum exp x; entropy -sum p log p; the `top` largest, ties to the lowest index.  A negative token has
             log probability 0.  Gradient of sum g lp + e H: p (-g - e (log p + H)), and g more at the token.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _rotate(name, tokens, heads, kv_heads, dim, rotary, axes, interleaved, train, dtype):
    return {"name": name, "kind": "rotate", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "axes": axes,
            "interleaved": interleaved, "train": train, "dtype": dtype}


def _append(name, tokens, heads, kv_heads, dim, rotary, axes, interleaved, bits, page, dtype):
    return {"name": name, "kind": "append", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "axes": axes,
            "interleaved": interleaved, "bits": bits, "page": page, "dtype": dtype}


def _attend(name, batch, longest, shortest, window, sinks, heads, kv_heads, dim, bits, page, dtype):
    return {"name": name, "kind": "attend", "batch": batch, "longest": longest, "shortest": shortest, "window": window, "sinks": sinks, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "bits": bits, "page": page, "dtype": dtype}


def _log_probs(name, rows, vocab, top, entropy, train, dtype):
    return {"name": name, "kind": "log_probs", "rows": rows, "vocab": vocab, "top": top, "entropy": entropy, "train": train, "dtype": dtype}


def listed():
    return [
        # A decode step of a few requests: the smallest call, where latency is all there is.
        _rotate("rotate_3tok", 3, 32, 8, 128, 128, 1, False, False, "fp16"),
        # Fine-tuning, forward and backward, a ragged batch; a quarter of each head is rotated, neighbours in pairs.
        _rotate("rotate_train_2043tok_r32_bf16", 2043, 32, 8, 128, 32, 1, True, True, "bf16"),
        # A batch of images and text: time, height and width, forward and backward.
        _rotate("rotate_train_16384tok_3axes_bf16", 16384, 32, 8, 128, 128, 3, False, True, "bf16"),
        # A decode batch: its queries rotated, its new rows written (and read back).
        _append("append_61tok_w4", 61, 32, 8, 128, 128, 1, False, 4, 16, "fp16"),
        # A chunk of a prompt with an image; 12 heads of 64.
        _append("append_509tok_3axes_w8_bf16", 509, 12, 12, 64, 64, 3, False, 8, 16, "bf16"),
        # The largest prompt, at once.
        _append("append_16384tok_w4_bf16", 16384, 32, 8, 128, 128, 1, False, 4, 32, "bf16"),
        # One short sequence of a model with 12 heads of 64.
        _attend("attend_1x203_last64_d64_w8", 1, 203, 203, 64, 4, 12, 12, 64, 8, 16, "fp16"),
        # Ordinary serving: 16 requests of any length up to 8192, the last 1000 tokens and four sinks.
        _attend("attend_16x8192_last1000_w4", 16, 8192, 1, 1000, 4, 32, 8, 128, 4, 16, "fp16"),
        # A full batch of very long conversations, whose caches hold a window each.
        _attend("attend_64x131071_last4096_w8_bf16", 64, 131071, 4096, 4096, 64, 32, 8, 128, 8, 64, "bf16"),
        # One sampled token of a small model, with five alternatives.
        _log_probs("log_probs_1x50272_top5", 1, 50272, 5, True, False, "fp16"),
        # A decode batch of a large vocabulary (odd, so that rows start anywhere), with twenty alternatives.
        _log_probs("log_probs_61x131071_top20_bf16", 61, 131071, 20, True, False, "bf16"),
        # The largest: the loss of a training batch with an entropy term, and its gradient.
        _log_probs("log_probs_train_8192x131072_bf16", 8192, 131072, 0, True, True, "bf16"),
    ]


def _log(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    kind = rng.choice(("rotate", "append", "attend", "log_probs"))
    dtype = rng.choice(("fp16", "bf16", "fp32" if kind != "attend" else "bf16"))
    if kind == "log_probs":
        train = rng.random() < 0.4
        vocab = _log(rng, 1000, 131072)
        rows = _log(rng, 1, max(1, min(8192, 8192 * 131072 // vocab // (2 if dtype == "fp32" else 1))))
        top = 0 if train else rng.choice((0, 1, 5, 20, 32))
        if top:
            rows = min(rows, max(1, 2 ** 28 // vocab))
        return _log_probs(None, rows, vocab, top, rng.random() < 0.6, train, dtype)
    kv_heads = _log(rng, 1, 32)
    heads = kv_heads * rng.choice((1, 2, 4, 5, 7, 8))
    if kind == "attend":
        dim, bits, page = rng.choice((64, 128, 128, 256)), rng.choice((2, 4, 4, 8)), rng.choice((16, 32, 48, 64))
        batch = _log(rng, 1, 96)
        longest = _log(rng, 1, 131072)
        sinks = rng.choice((0, 1, 4, 4, 64))
        # (visible tokens of all sequences: those of the largest listed case, 64 x 4160 of 8 heads of 128 in 8 bits, or fewer)
        window = _log(rng, 1, max(1, min(8192, 2.6e5 * 8 * 128 // (batch * kv_heads * dim))))
        return _attend(None, batch, longest, rng.randint(0, longest), window, sinks, heads, kv_heads, dim, bits, page, dtype)
    dim = rng.choice((64, 128, 128, 256))
    rotary, axes, interleaved = rng.choice((dim, dim, dim // 2, dim // 4)), rng.choice((1, 1, 2, 3)), rng.random() < 0.3
    tokens = _log(rng, 1, max(2, min(16384, 16384 * 40 * 128 // ((heads + kv_heads) * dim * (2 if dtype == "fp32" else 1)))))
    if kind == "rotate":
        return _rotate(None, tokens, heads, kv_heads, dim, rotary, axes, interleaved, rng.random() < 0.5, dtype)
    return _append(None, tokens, heads, kv_heads, dim, rotary, axes, interleaved, rng.choice((2, 4, 4, 8)), rng.choice((16, 32, 48, 64)), dtype)


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(shape, g, dtype):
    """Queries, keys or values: about N(0, 1), with channels that are larger or off zero, as projections give them."""
    x = torch.randn(shape, generator=g, device="cuda")
    x *= 0.5 + torch.rand(shape[-1], generator=g, device="cuda")
    x += 0.3 * torch.randn(shape[-1], generator=g, device="cuda")
    return x.to(dtype)


POSITIONS = 20480          # of the table of cosines and sines


def _sections(pairs, axes):
    """Pairs of each axis: a quarter of them time, the rest height and width."""
    if axes == 1:
        return (pairs,)
    if axes == 2:
        return (pairs // 2, pairs - pairs // 2)
    first, second = pairs // 4, (pairs - pairs // 4) // 2
    return (first, second, pairs - first - second)


def _frequencies(rotary):
    return 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)


def _positions(case, seed):
    """[axes, tokens] or, of one axis, [tokens]: decode steps anywhere, or a prompt from some offset on; of several axes text with images in it."""
    c = torch.Generator()
    c.manual_seed(seed * 1000003 + 31)
    n, axes = case["tokens"], case["axes"]
    if n <= 64:
        p = torch.randint(0, POSITIONS, (n,), generator=c)
    else:
        p = torch.arange(n) + int(torch.randint(0, POSITIONS - n + 1, (1,), generator=c))
    if axes == 1:
        return p
    all_axes = p.repeat(axes, 1)
    image = torch.arange(n) % 1000 >= 300              # of each thousand tokens the last 700 are a picture of 28 columns
    at = torch.arange(n) % 1000 - 300
    all_axes[-1][image] = (p[image] + at[image] % 28) % POSITIONS
    all_axes[-2][image] = (p[image] + at[image] // 28) % POSITIONS
    return all_axes


def _lengths(case, seed):
    """The sequences' lengths: the longest is there, and the shortest (0 only where it was drawn)."""
    c = torch.Generator()
    c.manual_seed(seed * 1000003 + 17)
    n = torch.randint(case["shortest"], case["longest"] + 1, (case["batch"],), generator=c)
    n[0] = case["longest"]
    if case["batch"] > 1:
        n[-1] = case["shortest"]
    return n


def _empty_cache(pages, case):
    h, s, words = case["kv_heads"], case["page"], case["dim"] * case["bits"] // 32
    return (torch.zeros((pages, h, s, words), dtype=torch.int32, device="cuda"), torch.zeros((pages, h, s, words), dtype=torch.int32, device="cuda"),
            torch.zeros((pages, h, s, 4), dtype=torch.float16, device="cuda"))


def _values(packed, params, bits, i):
    """fp32 values of rows: scale * (code - zero).  packed [..., words] int32, params [..., 4], i the first of its two constants."""
    shifts = torch.arange(0, 32, bits, device=packed.device, dtype=torch.int32)
    codes = ((packed[..., None] >> shifts) & (2 ** bits - 1)).flatten(-2).float()
    p = params.float()
    return p[..., i, None] * (codes - p[..., i + 1, None])


def _quantised(x, bits):
    """(packed words, scale, zero) of the rows of x (fp32)."""
    lo, hi = x.amin(-1).clamp(max=0.0), x.amax(-1).clamp(min=0.0)
    most = torch.full_like(hi, 2 ** bits - 1)
    exact = (hi - lo) / most
    scale = exact.half()
    scale = torch.where(scale.float() < exact, (scale.view(torch.int16) + 1).view(torch.float16), scale)
    scale = torch.maximum(scale, torch.full_like(scale, 2.0 ** -24))
    s = scale.float()
    zero = torch.round(-lo / s)
    codes = torch.clamp(torch.round(x / s[..., None] + zero[..., None]), 0, 2 ** bits - 1).to(torch.int32)
    shifts = torch.arange(0, 32, bits, device=x.device, dtype=torch.int32)
    words = (codes.unflatten(-1, (-1, 32 // bits)) << shifts).sum(-1, dtype=torch.int32)
    return words, scale, zero.half()


def _write(state, k, v, slots):
    kc, vc, params = state["k_codes"], state["v_codes"], state["params"]
    page, at = slots // state["page"], slots % state["page"]
    words, scale, zero = _quantised(k, state["bits"])
    kc[page, :, at] = words
    params[page, :, at, 0] = scale
    params[page, :, at, 1] = zero
    words, scale, zero = _quantised(v, state["bits"])
    vc[page, :, at] = words
    params[page, :, at, 2] = scale
    params[page, :, at, 3] = zero


def _read(state, slots):
    page, at = slots // state["page"], slots % state["page"]
    p = state["params"][page, :, at]
    return _values(state["k_codes"][page, :, at], p, state["bits"], 0), _values(state["v_codes"][page, :, at], p, state["bits"], 2)


def prepare(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    state = {"kind": case["kind"], "dtype": dtype}
    if case["kind"] == "log_probs":
        rows, vocab = case["rows"], case["vocab"]
        c = torch.Generator()
        c.manual_seed(seed * 1000003 + 37)
        logits = torch.empty((rows, vocab), dtype=dtype, device="cuda")
        for part in logits.split(max(1, (1 << 27) // vocab)):
            part.copy_(2.5 * torch.randn(part.shape, generator=g, device="cuda"))
        tokens = torch.randint(0, vocab, (rows,), generator=c)
        logits[torch.arange(rows, device="cuda"), tokens.cuda()] += 6.0          # (a model that often expects what comes)
        if case["train"] and rows > 8:
            tokens[torch.rand(rows, generator=c) < 0.1] = -100                    # padding
        state |= {"logits": logits, "tokens": tokens.cuda(), "top": case["top"], "entropy": case["entropy"], "train": case["train"]}
        if case["train"]:
            logits.requires_grad_()
            state["grad"] = torch.full((rows,), -1.0 / rows, device="cuda")
            state["grad_entropy"] = torch.full((rows,), -0.01 / rows, device="cuda") if case["entropy"] else None
        return state
    if case["kind"] == "attend":
        lengths, page, longest = _lengths(case, seed), case["page"], case["longest"]
        b, wide = case["batch"], -(-longest // page)
        # Pages that hold a visible token, in any order; the others are given up.
        at = torch.arange(wide)
        first = (lengths - case["window"]).clamp(min=0)
        held = (at < (lengths[:, None] + page - 1) // page) & ((at * page < case["sinks"]) | (at >= first[:, None] // page))
        pages = int(held.sum())
        order = torch.randperm(pages, generator=g, device="cuda").cpu()
        table = torch.full((b, wide), -1)
        table[held] = order
        state |= {"page": page, "bits": case["bits"], "window": case["window"], "sinks": case["sinks"],
                  "table": table.to(torch.int32).cuda(), "lengths": lengths.to(torch.int32).cuda()}
        state["k_codes"], state["v_codes"], state["params"] = _empty_cache(max(1, pages), case)
        for t in torch.arange(pages * page, device="cuda").split(max(1, (1 << 24) // (case["kv_heads"] * case["dim"]))):
            shape = (t.numel(), case["kv_heads"], case["dim"])
            _write(state, _rows(shape, g, dtype).float(), _rows(shape, g, dtype).float(), t)
        state["q"] = torch.randn((b, case["heads"], case["dim"]), generator=g, device="cuda").to(dtype)
        if own:
            from bitween_b200 import QuantizedKVCache
            state["cache"] = QuantizedKVCache.from_tensors(state["k_codes"], state["v_codes"], state["params"], case["bits"])
        return state
    n, heads, kv, dim, pairs = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["rotary"] // 2
    sections = _sections(pairs, case["axes"])
    angles = torch.arange(POSITIONS, dtype=torch.float64, device="cuda")[:, None] * _frequencies(case["rotary"]).cuda()
    state |= {"rotary": case["rotary"], "interleaved": case["interleaved"], "positions": _positions(case, seed).cuda(), "cos": angles.cos().float(), "sin": angles.sin().float(),
              "axis": torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).cuda(),
              "train": case.get("train", False)}
    fused = _rows((n, heads + 2 * kv, dim), g, dtype)                             # one projection gives all three
    state["q"], state["k"], state["v"] = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
    if state["train"]:
        state["q"], state["k"] = (x.contiguous().requires_grad_() for x in (state["q"], state["k"]))
        state["grad_q"], state["grad_k"] = (torch.randn(x.shape, generator=g, device="cuda").to(dtype) for x in (state["q"], state["k"]))
    if case["kind"] == "append":
        page = case["page"]
        wide = -(-n // page)
        pages = wide + wide // 4 + 1
        table = torch.randperm(pages, generator=g, device="cuda")[:wide]
        state |= {"page": page, "bits": case["bits"], "slots": (table[:, None] * page + torch.arange(page, device="cuda")).view(-1)[:n].contiguous()}
        state["k_codes"], state["v_codes"], state["params"] = _empty_cache(pages, case)
    if own:
        from bitween_b200 import QuantizedKVCache, RotaryPositions
        state["table"] = RotaryPositions(case["rotary"], POSITIONS, inv_freq=_frequencies(case["rotary"]), sections=None if case["axes"] == 1 else sections,
                                         interleaved=case["interleaved"])
        if case["kind"] == "append":
            state["cache"] = QuantizedKVCache.from_tensors(state["k_codes"], state["v_codes"], state["params"], case["bits"])
    return state


def _turned(state, x, back=False):
    """fp32 rows of x, rotated; or turned back."""
    p, pairs, x = state["positions"], state["rotary"] // 2, x.float()
    if p.dim() == 1:
        c, s = state["cos"][p], state["sin"][p]
    else:
        at = p[state["axis"]].T                                                    # [tokens, pairs]
        c, s = state["cos"].gather(0, at), state["sin"].gather(0, at)
    c, s = c[:, None], (-s if back else s)[:, None]
    if state["interleaved"]:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
    y1, y2 = a * c - b * s, b * c + a * s
    y = torch.stack((y1, y2), -1).flatten(-2) if state["interleaved"] else torch.cat((y1, y2), -1)
    return torch.cat((y, x[..., 2 * pairs:]), -1)


def _plain_attend(state):
    q, page = state["q"].float(), state["page"]
    b, heads, d = q.shape
    n, longest = state["lengths"].long()[:, None], state["table"].shape[1] * page
    # The visible places of each sequence: its sinks, then its window behind them.
    sinks, window = min(state["sinks"], longest), min(state["window"], longest)
    first = torch.arange(sinks, device=q.device).expand(b, -1)
    last = n - window + torch.arange(window, device=q.device)
    at = torch.cat((first, last), 1)
    seen = torch.cat((first < n, last >= sinks), 1)
    at = at.clamp(min=0)
    slot = state["table"].long().gather(1, at // page).clamp(min=0)
    at = at % page
    p = state["params"][slot, :, at].transpose(1, 2)                               # [B, Hkv, T, 4]
    k = _values(state["k_codes"][slot, :, at].transpose(1, 2), p, state["bits"], 0)
    kv = k.shape[1]
    s = (q.view(b, kv, heads // kv, d) / math.sqrt(d)) @ k.transpose(-1, -2)
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    w = torch.exp(s - m.masked_fill(m == -math.inf, 0.0))
    w = w / w.sum(-1, keepdim=True).clamp(min=1e-30)
    del k, s
    out = w @ _values(state["v_codes"][slot, :, at].transpose(1, 2), p, state["bits"], 2)
    return out.reshape(b, heads, d).to(state["dtype"])


def _plain_log_probs(state):
    x, t = state["logits"].detach().float(), state["tokens"]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    log_p = (x - m) - torch.log(total)
    there = t >= 0
    at = t.clamp(min=0)[:, None]
    out = {"log_probs": torch.where(there, log_p.gather(1, at)[:, 0], 0.0)}
    entropy = None
    if state["entropy"]:
        entropy = -(torch.exp(log_p) * log_p).sum(-1)
        out["entropy"] = entropy
    if state["top"]:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :state["top"]]
        out |= {"top_log_probs": log_p.gather(1, order), "top_tokens": order}
    if state["train"]:
        p = e.div_(total)
        g = torch.where(there, state["grad"], 0.0)[:, None]
        factor = -g
        if entropy is not None:
            factor = log_p.add_(entropy[:, None]).mul_(-state["grad_entropy"][:, None]).sub_(g)
        grad = p.mul_(factor)
        grad.scatter_add_(1, at, g)
        out["grad"] = grad.to(state["dtype"])
    return out


def run(state):
    kind = state["kind"]
    if kind == "attend":
        if own:
            return state["cache"].attend(state["q"], state["table"], state["lengths"], window=state["window"], sinks=state["sinks"])
        return _plain_attend(state)
    if kind == "append":
        if own:
            q = state["cache"].append_rotated(state["q"], state["k"], state["v"], state["slots"], state["table"], state["positions"])
            k, v = state["cache"].read(state["slots"], dtype=state["dtype"])
        else:
            q = _turned(state, state["q"]).to(state["dtype"])
            _write(state, _turned(state, state["k"]), state["v"].float(), state["slots"])
            k, v = (x.to(state["dtype"]) for x in _read(state, state["slots"]))
        return {"q": q, "k": k, "v": v}
    if kind == "rotate":
        if own:
            q, k = state["table"].rotate(state["positions"], state["q"], state["k"])
            if not state["train"]:
                return {"q": q, "k": k}
            dq, dk = torch.autograd.grad((q, k), (state["q"], state["k"]), (state["grad_q"], state["grad_k"]))
            return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
        out = {"q": _turned(state, state["q"].detach()), "k": _turned(state, state["k"].detach())}
        if state["train"]:
            out |= {"dq": _turned(state, state["grad_q"], back=True), "dk": _turned(state, state["grad_k"], back=True)}
        return {name: x.to(state["dtype"]) for name, x in out.items()}
    if not own:
        return _plain_log_probs(state)
    from bitween_b200 import token_log_probs
    r = token_log_probs(state["logits"], state["tokens"], entropy=state["entropy"], top=state["top"])
    out = {"log_probs": r.log_probs.detach()}
    if state["entropy"]:
        out["entropy"] = r.entropy.detach()
    if state["top"]:
        out |= {"top_log_probs": r.top_log_probs.detach(), "top_tokens": r.top_tokens}
    if state["train"]:
        outputs, grads = ((r.log_probs, r.entropy), (state["grad"], state["grad_entropy"])) if state["entropy"] else ((r.log_probs,), (state["grad"],))
        out["grad"] = torch.autograd.grad(outputs, state["logits"], grads)[0]
    return out


def _visible(case):
    """Tokens that a case's sequences show in the mean over lengths from the shortest to the longest."""
    most, lo, hi = case["window"] + case["sinks"], case["shortest"], case["longest"]
    seen = lambda n: min(n, most)  # noqa: E731
    if case["batch"] == 1:
        return seen(hi)
    under, width = min(max(most - lo, 0), hi - lo), max(1, hi - lo)
    mean = (under * (lo + lo + under) / 2 + (width - under) * most) / width if hi > lo else seen(hi)
    return seen(hi) + seen(lo) + (case["batch"] - 2) * mean


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "attend":
        tokens, h = _visible(case), case["heads"] * case["dim"]
        row = 2 * case["dim"] * case["bits"] / 8 + 8
        return {"bytes": int(tokens * case["kv_heads"] * row + 4 * case["batch"] * h), "flops": int(4 * tokens * h)}
    if case["kind"] == "log_probs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size * (3 if case["train"] else 1) + 16 * case["rows"], "flops": n * (12 if case["train"] else 5)}
    n, q, kv = case["tokens"], case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    table = n * (case["rotary"] // 2 * 8 + 8 * case["axes"])
    if case["kind"] == "rotate":
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * n * (q + kv) * size + table), "flops": passes * 3 * n * (case["heads"] + case["kv_heads"]) * case["rotary"]}
    row = case["kv_heads"] * (2 * case["dim"] * case["bits"] / 8 + 8)
    return {"bytes": int(2 * n * q * size + 4 * n * kv * size + n * row + table), "flops": 3 * n * (case["heads"] + case["kv_heads"]) * case["rotary"] + 8 * n * kv}


def exact(case, seed):
    """From the definitions, in 64 bits."""
    state = prepare(case, seed)
    if case["kind"] == "attend":
        out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
        group = case["heads"] // case["kv_heads"]
        shifts = torch.arange(0, 32, case["bits"], device="cuda")
        for b, n in enumerate(state["lengths"].tolist()):
            t = torch.arange(n, device="cuda")
            t = t[(t < case["sinks"]) | (t >= n - case["window"])]
            if not t.numel():
                continue
            page, at, both = state["table"][b].long()[t // case["page"]], t % case["page"], []
            for codes, i in ((state["k_codes"], 0), (state["v_codes"], 2)):
                c = (codes[page, :, at].long()[..., None] >> shifts).bitwise_and_(2 ** case["bits"] - 1).flatten(-2).double()
                p = state["params"][page, :, at].double()
                both.append(p[..., i, None] * (c - p[..., i + 1, None]))          # [T, Hkv, D]
            score = torch.einsum("hgd,thd->hgt", state["q"][b].double().view(-1, group, case["dim"]), both[0]) / math.sqrt(case["dim"])
            out[b] = torch.einsum("hgt,thd->hgd", torch.softmax(score, -1), both[1]).reshape(case["heads"], case["dim"])
        return out
    if case["kind"] == "log_probs":
        logits, tokens = state["logits"].detach(), state["tokens"]
        parts = []
        for lo in range(0, case["rows"], max(1, (1 << 28) // case["vocab"])):
            x, t = logits[lo:lo + max(1, (1 << 28) // case["vocab"])].double(), tokens[lo:lo + max(1, (1 << 28) // case["vocab"])]
            lp = torch.log_softmax(x, -1)
            del x
            rows = torch.arange(t.numel(), device="cuda")
            out = {"log_probs": torch.where(t >= 0, lp[rows, t.clamp(min=0)], 0.0)}
            h = torch.special.entr(lp.exp()).sum(-1)
            if case["entropy"]:
                out["entropy"] = h
            if case["top"]:
                out["top_log_probs"] = lp.topk(case["top"], -1).values
            if case["train"]:
                e = -0.01 / case["rows"] if case["entropy"] else 0.0
                g = torch.where(t >= 0, -1.0 / case["rows"], 0.0)[:, None].double()
                grad = lp.exp() * (-g - e * (lp + h[:, None]))
                grad[rows, t.clamp(min=0)] += g[:, 0]
                out["grad"] = grad.to(torch.float32)                              # (8 GB in 64 bits; the kernels' are 16-bit or fp32)
            parts.append(out)
        return {name: torch.cat([p[name] for p in parts]) for name in parts[0]} | ({"top_tokens": None} if case["top"] else {})
    freq = _frequencies(case["rotary"]).cuda()
    p = state["positions"].double()
    angle = (p[None] if p.dim() == 1 else p)[state["axis"]].T * freq              # [tokens, pairs]
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def turned(x, by):
        x, r = x.double(), case["rotary"]
        z = torch.view_as_complex(x[..., :r].unflatten(-1, (-1, 2)).contiguous()) if case["interleaved"] else torch.complex(x[..., :r // 2], x[..., r // 2:r])
        z = z * by
        y = torch.view_as_real(z).flatten(-2) if case["interleaved"] else torch.cat((z.real, z.imag), -1)
        return torch.cat((y, x[..., r:]), -1)

    out = {"q": turned(state["q"].detach(), turn)}
    k = turned(state["k"].detach(), turn)
    if case["kind"] == "rotate":
        out["k"] = k
        if case["train"]:
            out |= {"dq": turned(state["grad_q"], turn.conj()), "dk": turned(state["grad_k"], turn.conj())}
        return out
    most = 2 ** case["bits"] - 1
    for name, x in (("k", k), ("v", state["v"].double())):
        span = (x.amax(-1).clamp(min=0) - x.amin(-1).clamp(max=0)) / most
        down = span.half()
        step = 2.0 ** (torch.floor(torch.log2(down.double().clamp(min=2.0 ** -14))) - 10)
        s = (down.double() + step * (down.double() < span)).clamp(min=2.0 ** -24)[..., None]
        z = torch.round(-x.amin(-1, keepdim=True).clamp(max=0) / s)
        out[name] = s * (torch.round(x / s + z).clamp(0, most) - z)
    return out
