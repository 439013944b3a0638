"""The operators beside the packed linears, as cases that can be timed: the quantised key-value cache (written, read back, attended to
by new tokens) and the low-rank adapters of many requests beside a shared projection.

Where `own` is false, `run` computes them in elementary torch operations in 32 bits; where it is true, it makes the calls of this
package.  The formulas:

  cache     a row is one token's D values of one head.  With Q = 2^bits - 1, lo = min(row, 0), hi = max(row, 0):
            scale = (hi - lo) / Q rounded up to fp16, at least 2^-24; zero = round(-lo / scale); code = clamp(round(x / scale + zero), 0, Q).
            A row stands for scale * (code - zero).  Codes are packed like weights: code i of word j is element j * 32 / bits + i.
  attend    out[b, h] = sum_t softmax_t(q[b, h] . K[t, h / group] / sqrt(D)) V[t, h / group] over the t < lengths[b] of a paged cache
  adapters  y[t] = base[t] + scaling[i] * up[i]^T (down[i] x[t]) with i = index[t]; -1 stands for no adapter
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _attend(name, batch, longest, shortest, heads, kv_heads, dim, bits, page, dtype):
    return {"name": name, "kind": "attend", "batch": batch, "longest": longest, "shortest": shortest, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "bits": bits, "page": page, "dtype": dtype}


def _chunk(name, new, prefix, kv_heads, dim, bits, page, dtype):
    return {"name": name, "kind": "chunk", "new": new, "prefix": prefix, "kv_heads": kv_heads, "dim": dim, "bits": bits, "page": page, "dtype": dtype}


def _adapters(name, kind, tokens, adapters, rank, cols, rows, dtype):
    return {"name": name, "kind": kind, "tokens": tokens, "adapters": adapters, "rank": rank, "cols": cols, "rows": rows, "dtype": dtype}


def listed():
    return [
        # One short sequence of a model with 12 heads of 64: the smallest call, where latency is all there is.
        _attend("attend_1x49_d64_w8", 1, 49, 49, 12, 12, 64, 8, 16, "fp16"),
        # Ordinary serving: 16 requests of any length up to 2048, grouped queries, 4 bits.
        _attend("attend_16x2048_w4", 16, 2048, 1, 32, 8, 128, 4, 16, "fp16"),
        # A full batch of long conversations.
        _attend("attend_64x8192_w4_bf16", 64, 8192, 4096, 32, 8, 128, 4, 32, "bf16"),
        # One very long document, an odd length: the work has to be split over the cache's length.
        _attend("attend_1x131071_w8_bf16", 1, 131071, 131071, 32, 8, 128, 8, 64, "bf16"),
        # The new rows of a decode batch, written and read back.
        _chunk("rows_37_w8", 37, 0, 8, 128, 8, 16, "fp16"),
        # A chunk of a prompt is appended, then the whole prefix is read back for the prompt's attention.
        _chunk("chunk_509_of_4093_w4", 509, 3584, 8, 128, 4, 16, "bf16"),
        # The largest prompt, written at once.
        _chunk("chunk_16384_w8", 16384, 0, 8, 128, 8, 32, "fp16"),
        # A few requests with adapters of their own beside a 4096 x 4096 projection.
        _adapters("adapters_5tok_r16", "adapters", 5, 3, 16, 4096, 4096, "fp16"),
        # A decode batch with many adapters beside the widest projection of a block.
        _adapters("adapters_61tok_r32_bf16", "adapters", 61, 24, 32, 4096, 14336, "bf16"),
        # A batch of prompts.
        _adapters("adapters_2043tok_r16", "adapters", 2043, 7, 16, 4096, 4096, "fp16"),
        # Fine-tuning, a short batch beside a narrow projection: forward and backward.
        _adapters("train_509tok_r8", "train", 509, 1, 8, 4096, 1024, "fp16"),
        # The largest: fine-tuning beside the widest projection.
        _adapters("train_8192tok_r64_bf16", "train", 8192, 2, 64, 4096, 14336, "bf16"),
    ]


def _log(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    kind = rng.choice(("attend", "attend", "chunk", "adapters", "train"))
    dtype = rng.choice(("fp16", "bf16"))
    if kind in ("attend", "chunk"):
        dim, bits, page = rng.choice((64, 128, 128, 256)), rng.choice((2, 4, 4, 8)), rng.choice((16, 32, 48, 64))
        kv_heads = _log(rng, 1, 32)
    if kind == "attend":
        heads = kv_heads * rng.choice((1, 2, 4, 5, 7, 8, 16))
        batch = _log(rng, 1, 96)
        # (cached tokens of all sequences: those of the largest listed case, 64 x 6144 of 8 heads of 128, or fewer)
        longest = _log(rng, 1, max(1, min(131072, 3.0e6 * 128 // (batch * kv_heads * dim))))
        return _attend(None, batch, longest, rng.randint(0, longest), heads, kv_heads, dim, bits, page, dtype)
    if kind == "chunk":
        most = max(2, min(16384, 16384 * 8 * 128 // (kv_heads * dim)))
        new = _log(rng, 1, most)
        return _chunk(None, new, rng.choice((0, _log(rng, 1, most))), kv_heads, dim, bits, page, dtype)
    cols, rows = 64 * _log(rng, 8, 224), 64 * _log(rng, 8, 224)
    rank = 8 * rng.choice((1, 2, 2, 4, 8))
    tokens = _log(rng, 1, max(2, min(8192, 8192 * 4096 * 14336 // (cols * rows))))
    adapters = _log(rng, 1, 32) if kind == "adapters" else _log(rng, 1, 4)
    return _adapters(None, kind, tokens, adapters, rank, cols, rows, dtype)


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(case, seed):
    """The sequences' lengths: the longest is there, and the shortest (0 only where it was drawn)."""
    c = torch.Generator()
    c.manual_seed(seed * 1000003 + 17)
    n = torch.randint(case["shortest"], case["longest"] + 1, (case["batch"],), generator=c)
    n[0] = case["longest"]
    if case["batch"] > 1:
        n[-1] = case["shortest"]
    return n


def _rows(shape, g, dtype):
    """Keys or values: about N(0, 1), with channels that are larger or off zero, as projections give them."""
    x = torch.randn(shape, generator=g, device="cuda")
    x *= 0.5 + torch.rand(shape[-1], generator=g, device="cuda")
    x += 0.3 * torch.randn(shape[-1], generator=g, device="cuda")
    return x.to(dtype)


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
    """(packed words, scale, zero) of the rows of x."""
    x = x.float()
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
    if case["kind"] in ("attend", "chunk"):
        state = {"kind": case["kind"], "page": case["page"], "bits": case["bits"], "dtype": dtype}
        if case["kind"] == "attend":
            lengths = _lengths(case, seed)
            wide = -(-case["longest"] // case["page"])
            pages = case["batch"] * wide
            table = torch.randperm(pages, generator=g, device="cuda").view(case["batch"], wide)
            state["k_codes"], state["v_codes"], state["params"] = _empty_cache(pages, case)
            lengths = lengths.cuda()
            held = torch.arange(wide * case["page"], device="cuda")[None] < lengths[:, None]
            slots = (table[:, :, None] * case["page"] + torch.arange(case["page"], device="cuda")).view(case["batch"], -1)
            cached = slots[held]
            state["table"], state["lengths"] = table.to(torch.int32), lengths.to(torch.int32)
            state["q"] = torch.randn((case["batch"], case["heads"], case["dim"]), generator=g, device="cuda").to(dtype)
        else:
            total = case["prefix"] + case["new"]
            wide = -(-total // case["page"])
            pages = wide + wide // 4 + 1
            table = torch.randperm(pages, generator=g, device="cuda")[:wide]
            slots = (table[:, None] * case["page"] + torch.arange(case["page"], device="cuda")).view(-1)[:total]
            state["k_codes"], state["v_codes"], state["params"] = _empty_cache(pages, case)
            cached = slots[:case["prefix"]]
            state["slots"], state["new"] = slots, slots[case["prefix"]:].contiguous()
            shape = (case["new"], case["kv_heads"], case["dim"])
            state["k"], state["v"] = _rows(shape, g, dtype), _rows(shape, g, dtype)
        for t in cached.split(max(1, (1 << 24) // (case["kv_heads"] * case["dim"]))):       # (temporaries of some hundred MB)
            shape = (t.numel(), case["kv_heads"], case["dim"])
            _write(state, _rows(shape, g, dtype), _rows(shape, g, dtype), t)
        if own:
            from bitween_b200 import QuantizedKVCache
            state["cache"] = QuantizedKVCache.from_tensors(state["k_codes"], state["v_codes"], state["params"], case["bits"])
        return state
    n, r, k, rows, t = case["adapters"], case["rank"], case["cols"], case["rows"], case["tokens"]
    c = torch.Generator()
    c.manual_seed(seed * 1000003 + 29)
    if t <= 64:     # decode: a token a request, in any order; some have no adapter
        index = torch.randint(-1 if t > n else 0, n, (t,), generator=c)
    else:           # prompts: runs of one adapter each, and a run that has none
        index = torch.randint(0, n, (t,), generator=c).sort().values
        if case["kind"] == "adapters" and n > 1:
            index = torch.where(index == n // 2, -1, index)
    state = {"kind": case["kind"], "index": index.to(torch.int32).cuda(),
             "x": torch.randn((t, k), generator=g, device="cuda").to(dtype),
             "down": (torch.randn((n, r, k), generator=g, device="cuda") / math.sqrt(k)).to(dtype),
             "up": (0.1 * torch.randn((n, r, rows), generator=g, device="cuda")).to(dtype),
             "scaling": 0.5 + torch.rand((n,), generator=g, device="cuda"),
             "base": torch.randn((t, rows), generator=g, device="cuda").to(dtype)}
    if case["kind"] == "train":
        state["grad"] = torch.randn((t, rows), generator=g, device="cuda").to(dtype)
        for name in ("x", "down", "up"):
            state[name].requires_grad_()
    return state


def _plain_attend(state):
    q, page = state["q"].float(), state["page"]
    b, heads, d = q.shape
    at = state["table"].long()
    p = state["params"][at].transpose(1, 2).flatten(2, 3)                       # [B, Hkv, T, 4]
    k = _values(state["k_codes"][at].transpose(1, 2).flatten(2, 3), p, state["bits"], 0)
    kv = k.shape[1]
    s = (q.view(b, kv, heads // kv, d) / math.sqrt(d)) @ k.transpose(-1, -2)
    held = torch.arange(at.shape[1] * page, device=q.device)[None] < state["lengths"][:, None]
    s = s.masked_fill(~held[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    w = torch.exp(s - m.masked_fill(m == -math.inf, 0.0))
    w = w / w.sum(-1, keepdim=True).clamp(min=1e-30)
    del k, s
    out = w @ _values(state["v_codes"][at].transpose(1, 2).flatten(2, 3), p, state["bits"], 2)
    return out.reshape(b, heads, d).to(state["dtype"])


def _plain_adapters(state):
    x, down, up = state["x"].detach().float(), state["down"].detach().float(), state["up"].detach().float()
    n, r = down.shape[:2]
    chosen = (state["index"][:, None] == torch.arange(n, device=x.device)) * state["scaling"]     # [T, n]: the factor of the token's adapter
    chosen = chosen.repeat_interleave(r, 1)
    h = (x @ down.flatten(0, 1).T) * chosen
    y = (state["base"].float() + h @ up.flatten(0, 1)).to(state["base"].dtype)
    if state["kind"] == "adapters":
        return y
    grad = state["grad"].float()
    dh = (grad @ up.flatten(0, 1).T) * chosen
    dx = dh @ down.flatten(0, 1)
    return {"y": y, "dx": dx.to(y.dtype), "ddown": (dh.T @ x).view_as(down).to(y.dtype), "dup": (h.T @ grad).view_as(up).to(y.dtype)}


def run(state):
    if state["kind"] == "attend":
        if own:
            return state["cache"].attend(state["q"], state["table"], state["lengths"])
        return _plain_attend(state)
    if state["kind"] == "chunk":
        if own:
            state["cache"].append(state["k"], state["v"], state["new"])
            k, v = state["cache"].read(state["slots"], dtype=state["dtype"])
        else:
            _write(state, state["k"], state["v"], state["new"])
            k, v = (x.to(state["dtype"]) for x in _read(state, state["slots"]))
        return {"k": k, "v": v}
    if not own:
        return _plain_adapters(state)
    from bitween_b200 import adapter_matmul
    y = adapter_matmul(state["x"], state["down"], state["up"], state["index"], scaling=state["scaling"], base=state["base"])
    if state["kind"] == "adapters":
        return y
    dx, ddown, dup = torch.autograd.grad(y, (state["x"], state["down"], state["up"]), state["grad"])
    return {"y": y.detach(), "dx": dx, "ddown": ddown, "dup": dup}


def _mean_tokens(case):
    """Tokens that a case's sequences hold in the mean: the longest and the shortest are there, the others are between."""
    b = case["batch"]
    mid = (case["longest"] + case["shortest"]) / 2
    return case["longest"] if b == 1 else case["longest"] + case["shortest"] + (b - 2) * mid


def work(case):
    if case["kind"] == "attend":
        tokens, h = _mean_tokens(case), case["heads"] * case["dim"]
        row = 2 * case["dim"] * case["bits"] / 8 + 8
        return {"bytes": int(tokens * case["kv_heads"] * row + 4 * case["batch"] * h), "flops": int(4 * tokens * h)}
    if case["kind"] == "chunk":
        values, row = case["kv_heads"] * 2 * case["dim"], case["kv_heads"] * (2 * case["dim"] * case["bits"] / 8 + 8)
        total = case["prefix"] + case["new"]
        return {"bytes": int(case["new"] * (2 * values + row) + case["prefix"] * row + total * 2 * values), "flops": 4 * total * values}
    t, k, n, r = case["tokens"], case["cols"], case["rows"], case["rank"]
    used = min(case["adapters"], t)
    weights = used * r * (k + n)
    passes = 1 if case["kind"] == "adapters" else 3
    elements = t * k + 2 * t * n + weights
    if case["kind"] == "train":          # and the gradient read, those of x and of the adapters written
        elements += t * n + t * k + case["adapters"] * r * (k + n)
    return {"bytes": 2 * elements, "flops": passes * 2 * t * r * (k + n)}


def exact(case, seed):
    """From the definitions, in 64 bits."""
    state = prepare(case, seed)
    if case["kind"] == "attend":
        if case["batch"] * case["longest"] * case["kv_heads"] * case["dim"] > 64 * 8192 * 8 * 128:
            return None
        out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
        group = case["heads"] // case["kv_heads"]
        shifts = torch.arange(0, 32, case["bits"], device="cuda")
        for b, n in enumerate(state["lengths"].tolist()):
            if n == 0:
                continue
            pages = state["table"][b, :-(-n // case["page"])].long()
            both = []
            for codes, at in ((state["k_codes"], 0), (state["v_codes"], 2)):
                c = (codes[pages].long()[..., None] >> shifts).bitwise_and_(2 ** case["bits"] - 1).flatten(-2).double()
                p = state["params"][pages].double()
                both.append((p[..., at, None] * (c - p[..., at + 1, None])).permute(1, 0, 2, 3).flatten(1, 2)[:, :n])
            score = torch.einsum("hgd,htd->hgt", state["q"][b].double().view(-1, group, case["dim"]), both[0]) / math.sqrt(case["dim"])
            out[b] = torch.einsum("hgt,htd->hgd", torch.softmax(score, -1), both[1]).reshape(case["heads"], case["dim"])
        return out
    if case["kind"] == "chunk":
        most = 2 ** case["bits"] - 1

        def held(x):
            x = x.double()
            span = (x.amax(-1).clamp(min=0) - x.amin(-1).clamp(max=0)) / most
            down = span.half()
            step = 2.0 ** (torch.floor(torch.log2(down.double().clamp(min=2.0 ** -14))) - 10)
            s = (down.double() + step * (down.double() < span)).clamp(min=2.0 ** -24)[..., None]
            z = torch.round(-x.amin(-1, keepdim=True).clamp(max=0) / s)
            return s * (torch.round(x / s + z).clamp(0, most) - z)

        out = {}
        page, at = state["slots"] // case["page"], state["slots"] % case["page"]
        shifts = torch.arange(0, 32, case["bits"], device="cuda")
        for name, codes, i in (("k", state["k_codes"], 0), ("v", state["v_codes"], 2)):
            c = (codes[page, :, at].long()[..., None] >> shifts).bitwise_and_(most).flatten(-2).double()
            p = state["params"][page, :, at].double()
            out[name] = p[..., i, None] * (c - p[..., i + 1, None])
            out[name][case["prefix"]:] = held(state[name])
        return out
    x, down, up, f = (state[name].detach().double() for name in ("x", "down", "up", "scaling"))
    y, index = state["base"].double(), state["index"]
    grads = {"dx": torch.zeros_like(x), "ddown": torch.zeros_like(down), "dup": torch.zeros_like(up)}
    for i in range(case["adapters"]):
        mine = (index == i).nonzero()[:, 0]
        h = x[mine] @ down[i].T
        y[mine] += f[i] * (h @ up[i])
        if case["kind"] == "train":
            grad = state["grad"][mine].double()
            dh = f[i] * (grad @ up[i].T)
            grads["dx"][mine] = dh @ down[i]
            grads["ddown"][i] = dh.T @ x[mine]
            grads["dup"][i] = f[i] * (h.T @ grad)
    return y if case["kind"] == "adapters" else {"y": y, **grads}
