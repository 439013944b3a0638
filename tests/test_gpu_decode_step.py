"""Rotary positions, rotated appends, windowed attention and log probabilities as programs use them: together, under autograd, captured, on other streams, and
on both host paths."""
import math
import os
import subprocess
import sys
import threading

import pytest
import torch

from bitween_b200 import AdaptedLinear, QuantizedKVCache, QuantizedLinear, RotaryPositions, token_log_probs
from bitween_b200.kernels import _lib

DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_lib, "_operators", _lib._NoOperators)
    return request.param


def _packed(inner, outer, seed):
    lin = torch.nn.Linear(inner, outer, bias=False)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(outer, inner, generator=torch.Generator().manual_seed(seed)) * inner ** -0.5)
    return QuantizedLinear.from_float(lin.to(DEV), bits=8, group_size=64)


def test_calls_that_are_not_plain_are_left_to_the_python_path():
    ops = _lib.host_operators()
    codes, params = torch.zeros(2, 1, 16, 8, dtype=torch.int32), torch.zeros(2, 1, 16, 4).half()
    x, i64, i32 = torch.zeros(3, 1, 64).half(), torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int32)
    r = RotaryPositions(64, 10, device="cpu")
    assert ops.rotate(r.table, r._meta, i64, x) is None and ops.rotate(1, 2, 3, 4) is None and ops.rotate(r.table, r._meta, i64) is None
    assert ops.kv_append_rotated(codes, codes, params, 4, x, x, x, i64, r.table, r._meta, i64) is None and ops.kv_append_rotated(codes) is None
    assert ops.kv_attend(codes, codes, params, 4, x, i32[:, None], i32, 0.1, 5, 1) is None and ops.kv_attend(codes, codes, params, 4, x, i32[:, None], i32, 0.1, 1 << 80, -1) is None
    assert ops.token_log_probs(x, i64, True, 3) is None and ops.token_log_probs(x, None, 1, 3) is None and ops.token_log_probs(None, None, False, 0) is None


def _step(seed=1):
    """(rotary, cache, q, k, v, slots, positions, page table, lengths, logits, tokens) of a small batch."""
    g = _gen(seed)
    rotary = RotaryPositions(128, 400, sections=(16, 24, 24))
    cache = QuantizedKVCache(90, 16, 2, 128, bits=4, device=DEV)
    kv = torch.randn(90 * 16, 4, 128, generator=g, device=DEV).half()
    cache.append(kv[:, :2], kv[:, 2:], torch.arange(90 * 16, device=DEV))
    fused = torch.randn(5, 12, 128, generator=g, device=DEV).half()
    table = torch.randperm(90, generator=g, device=DEV)[:85].view(5, 17).to(torch.int32)
    lengths = torch.tensor([200, 1, 17, 272, 96], dtype=torch.int32, device=DEV)
    slots = table.long().gather(1, ((lengths - 1) // 16).long()[:, None])[:, 0] * 16 + (lengths.long() - 1) % 16
    positions = torch.randint(0, 400, (3, 5), generator=g, device=DEV)
    logits = 3 * torch.randn(5, 5001, generator=g, device=DEV)
    return rotary, cache, fused[:, :8], fused[:, 8:10], fused[:, 10:], slots, positions, table, lengths, logits, torch.randint(0, 5001, (5,), generator=g, device=DEV)


def _run(rotary, cache, q, k, v, slots, positions, table, lengths, logits, tokens):
    turned = cache.append_rotated(q, k, v, slots, rotary, positions)
    return [turned, *rotary.rotate(positions, q, k), cache.attend(turned, table, lengths, window=50, sinks=4), cache.attend(turned, table[:1, :3].expand(5, -1), lengths.clamp(max=40),
            softmax_scale=0.2, window=20), *cache.read(slots), *token_log_probs(logits, tokens, entropy=True, top=6), token_log_probs(logits.half(), tokens).log_probs]


@pytest.mark.gpu
def test_both_host_paths_are_alike(monkeypatch):
    args = _step()
    rotary, cache, q, k, v, slots, positions, table, lengths, logits, tokens = args
    ops = _lib.host_operators()
    for call in ((ops.rotate, rotary.table, rotary._meta, positions, q, k), (ops.rotate, rotary.table, rotary._meta, positions, q), (ops.rotate, rotary.table, rotary._meta, positions[0], q),
                 (ops.kv_append_rotated, *cache._cache, q, k, v, slots, rotary.table, rotary._meta, positions), (ops.kv_append_rotated, *cache._cache, None, k, v, slots, rotary.table, rotary._meta, positions[1]),
                 (ops.kv_attend, *cache._cache, q, table, lengths, 0.1, 50, 4), (ops.token_log_probs, logits, tokens, True, 6), (ops.token_log_probs, logits, None, False, 1)):
        assert call[0](*call[1:]) is not None
    for call in ((ops.rotate, rotary.table[:9], rotary._meta, positions, q), (ops.rotate, rotary.table, rotary._meta, positions.int(), q), (ops.rotate, rotary.table, rotary._meta, positions[:2], q),
                 (ops.rotate, rotary.table, rotary._meta, positions, q[..., :64]), (ops.rotate, rotary.table, rotary._meta, positions, q, k.float()), (ops.rotate, rotary.table, rotary._meta, positions, q[..., ::2]),
                 (ops.rotate, rotary.table, rotary._meta, positions.T.contiguous().T, q), (ops.rotate, rotary.table, (128, 0, 3, b"", 400), positions, q),
                 (ops.kv_append_rotated, *cache._cache, q.float(), k, v, slots, rotary.table, rotary._meta, positions), (ops.kv_append_rotated, *cache._cache, q, k, v, slots.int(), rotary.table, rotary._meta, positions),
                 (ops.kv_attend, *cache._cache, q, table, lengths, 0.1, -1, 4), (ops.kv_attend, *cache._cache, q, table, lengths.long(), 0.1, 4, 4),
                 (ops.token_log_probs, logits, tokens.int(), True, 6), (ops.token_log_probs, logits, tokens[:3], True, 6), (ops.token_log_probs, logits, tokens, True, 33),
                 (ops.token_log_probs, logits.double(), tokens, True, 3), (ops.token_log_probs, logits.T.contiguous().T, tokens, True, 3)):
        assert call[0](*call[1:]) is None, call[0]
    native = _run(*args)
    leaves = [t.clone().requires_grad_() for t in (q, k, logits)]

    def grads():
        yq, yk = rotary.rotate(positions, leaves[0], leaves[1])
        r = token_log_probs(leaves[2], tokens, entropy=True, top=6)
        names = {type(yq.grad_fn).__name__, type(r.entropy.grad_fn).__name__}
        w = [torch.randn(t.shape, generator=_gen(2), device=DEV).to(t.dtype) for t in (yq, yk, r.log_probs, r.entropy, r.top_log_probs)]
        return names, torch.autograd.grad((yq, yk, r.log_probs, r.entropy, r.top_log_probs), leaves, w)

    names, native_grads = grads()
    monkeypatch.setattr(_lib, "_operators", _lib._NoOperators)
    python = _run(*_step())
    assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(native, python))
    python_names, python_grads = grads()
    assert not names & python_names and all(torch.equal(a, b) for a, b in zip(native_grads, python_grads))


@pytest.mark.gpu
def test_a_decode_step_from_projections_to_answer():
    """Packed projections with an adapter a request, keys rotated into the cache, attention over a window and sinks, an output head, its log probabilities: a prompt token by token
    gives what the formulas give in 64 bits on the rows that the cache holds."""
    hidden, heads, kv_heads, dim, batch, steps, vocab, window, sinks = 512, 8, 2, 64, 3, 60, 1000, 20, 3
    layer = AdaptedLinear(_packed(hidden, (heads + 2 * kv_heads) * dim, 50), 2, 8)
    head = _packed(heads * dim, vocab, 51)
    with torch.no_grad():
        layer.up.copy_(torch.randn(layer.up.shape, generator=_gen(60), device=DEV) * 0.1)
    index = torch.tensor([0, -1, 1], dtype=torch.int32, device=DEV)
    rotary = RotaryPositions(32, 100, sections=(4, 6, 6))
    cache = QuantizedKVCache(13, 16, kv_heads, dim, bits=8, device=DEV)
    table = torch.tensor([[4, 1, 12, 11], [0, 7, 9, 2], [8, 3, 6, 5]], dtype=torch.int32, device=DEV)
    lengths = torch.zeros(batch, dtype=torch.int32, device=DEV)
    with torch.no_grad():
        for t in range(steps):
            x = torch.randn(batch, hidden, generator=_gen(70 + t), device=DEV).half()
            fused = layer(x, index).view(batch, heads + 2 * kv_heads, dim)
            q, k, v = fused[:, :heads], fused[:, heads:heads + kv_heads], fused[:, heads + kv_heads:]
            positions = torch.tensor([t, t // 3, t % 7], device=DEV)[:, None].expand(3, batch).contiguous()
            slots = table[:, t // 16].long() * 16 + t % 16
            q = cache.append_rotated(q, k, v, slots, rotary, positions)
            assert torch.equal(q, rotary.rotate(positions, fused[:, :heads]))
            lengths += 1
            a = cache.attend(q, table, lengths, window=window, sinks=sinks)
            logits = head(a.view(batch, heads * dim))
            answer = token_log_probs(logits, logits.argmax(-1), entropy=True, top=5)
    pos = torch.arange(steps, device=DEV)
    pos = pos[(pos < sinks) | (pos >= steps - window)]
    half = 2.0 ** -11
    for b in range(batch):
        k, v = (r.double().repeat_interleave(heads // kv_heads, 1) for r in cache.read(table[b, pos // 16].long() * 16 + pos % 16, dtype=torch.float32))
        w = torch.softmax(torch.einsum("hd,thd->ht", q[b].double(), k) * dim ** -0.5, -1)
        want, size = torch.einsum("ht,thd->hd", w, v), torch.einsum("ht,thd->hd", w, v.abs())
        assert bool(((a[b].double() - want).abs() <= half * want.abs() + 2.0 ** -14 * size + 2.0 ** -25).all())
    lp = torch.log_softmax(logits.double(), -1)
    assert torch.equal(answer.top_tokens[:, 0], logits.argmax(-1)) and torch.equal(answer.log_probs, answer.top_log_probs[:, 0])
    # (fp16 logits of some units: x - m is exact, and a sum of 1000 weights good to 2^-20)
    assert bool(((answer.top_log_probs.double() - lp.gather(1, answer.top_tokens)).abs() <= 2.0 ** -18).all())


@pytest.mark.gpu
def test_a_loss_trains_adapters_through_rotation_and_log_probabilities(path):
    """The gradient of a loss that goes through adapters, rotation, a product and token_log_probs: alike to that of the formulas in torch, whose elementary steps round elsewhere."""
    hidden, heads, dim, tokens, vocab = 128, 2, 64, 24, 300
    layer = AdaptedLinear(_packed(hidden, heads * dim, 80), 1, 8)
    with torch.no_grad():
        layer.up.copy_(torch.randn(layer.up.shape, generator=_gen(81), device=DEV) * 0.1)
    rotary = RotaryPositions(dim, 64)
    x = torch.randn(tokens, hidden, generator=_gen(82), device=DEV).half()
    index, positions = torch.zeros(tokens, dtype=torch.int32, device=DEV), torch.arange(tokens, device=DEV)
    out = torch.randn(heads * dim, vocab, generator=_gen(83), device=DEV).half() * 0.1
    target = torch.randint(0, vocab, (tokens,), generator=_gen(84), device=DEV)
    target[3] = -100

    def loss(own):
        y = layer(x, index).view(tokens, heads, dim)
        if own:
            logits = rotary.rotate(positions, y).flatten(1) @ out
            r = token_log_probs(logits, target, entropy=True)
            return -r.log_probs.sum() / 23 - 0.01 * r.entropy.mean()
        c, s = rotary.table[positions][:, None].unbind(-1)
        a, b = y.float().chunk(2, -1)
        logits = torch.cat((a * c - b * s, b * c + a * s), -1).half().flatten(1) @ out
        lp = torch.log_softmax(logits.float(), -1)
        at = torch.where(target >= 0, lp.gather(1, target.clamp(min=0)[:, None])[:, 0], 0.0)
        return -at.sum() / 23 + 0.01 * (lp.exp() * lp).sum(-1).mean()

    results = []
    for own in (True, False):
        layer.zero_grad()
        y = loss(own)
        y.backward()
        results.append((float(y), layer.down.grad.double(), layer.up.grad.double()))
    assert abs(results[0][0] - results[1][0]) <= 2.0 ** -17 * 8
    for a, b in zip(results[0][1:], results[1][1:]):
        # fp16 gradients between the steps, rounded at the same places of the same values or a step beside: 2^-11 each, at four places
        assert float((a - b).norm()) <= 2.0 ** -8 * float(b.norm()) and float(b.norm()) > 0


@pytest.mark.gpu
def test_gradients_cannot_be_differentiated_again_and_changed_tensors_are_noticed(path):
    rotary, cache, q, k, v, slots, positions, table, lengths, logits, tokens = _step()
    q, logits = q.clone().requires_grad_(), logits.clone().requires_grad_()
    for call, leaf in ((lambda: rotary.rotate(positions, q), q), (lambda: token_log_probs(logits, tokens).log_probs, logits)):
        y = call()
        grad = torch.ones_like(y, requires_grad=True)
        want = torch.autograd.grad(y, leaf, grad.detach(), retain_graph=True)[0]
        got = torch.autograd.grad(y, leaf, grad, create_graph=True)[0]
        assert torch.equal(got.detach(), want)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            got.float().sum().backward()
    for changed, call in ((positions, lambda: rotary.rotate(positions, q)), (rotary.table, lambda: rotary.rotate(positions, q)), (tokens, lambda: token_log_probs(logits, tokens).log_probs)):
        y = call()
        changed.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    y = token_log_probs(logits * 1.0, tokens - 1, top=3)
    y.top_tokens.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.top_log_probs.sum().backward()


@pytest.mark.gpu
def test_saved_tensors_that_hooks_give_back(path):
    rotary, cache, q, k, v, slots, positions, table, lengths, logits, tokens = _step()
    q, logits = q.clone().requires_grad_(), logits.clone().requires_grad_()

    def grads():
        r = token_log_probs(logits, tokens, entropy=True, top=3)
        return torch.autograd.grad((rotary.rotate(positions, q).float().sum() + r.log_probs.sum() + r.top_log_probs[:, 1].sum() + r.entropy[2]), (q, logits))

    want = grads()
    with torch.autograd.graph.save_on_cpu():
        assert all(torch.equal(a, b) for a, b in zip(grads(), want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.clone().T.contiguous().T if t.dim() == 2 else t):
        assert all(torch.equal(a, b) for a, b in zip(grads(), want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:1] if t.dtype == torch.int64 else t):
        with pytest.raises(RuntimeError, match="hooks"):
            grads()


@pytest.mark.gpu
def test_modes_subclasses_and_other_streams():
    args = _step()
    want = _run(*args)
    rotary, cache, q, k, v, slots, positions, table, lengths, logits, tokens = args

    class Sub(torch.Tensor):
        pass

    ops = _lib.host_operators()
    assert ops.rotate(rotary.table, rotary._meta, positions, q.as_subclass(Sub)) is None and ops.token_log_probs(logits.as_subclass(Sub), tokens, False, 0) is None
    assert torch.equal(rotary.rotate(positions, q.as_subclass(Sub)).as_subclass(torch.Tensor), want[1])
    assert torch.equal(token_log_probs(logits.as_subclass(Sub), tokens).log_probs.as_subclass(torch.Tensor), want[7])
    z = torch.complex(torch.zeros_like(logits), -logits).conj().imag                  # a view with a pending negation
    assert z.is_neg() and torch.equal(token_log_probs(z, tokens).log_probs, want[7])
    assert torch.equal(rotary.rotate(positions, torch.complex(torch.zeros(q.shape, device=DEV), -q.float()).conj().imag), rotary.rotate(positions, q.float()))
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(_run(*args), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(*args)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    wrong = []

    def work():
        for _ in range(20):
            if not all(torch.equal(a, b) for a, b in zip(_run(*args), want)):
                wrong.append(1)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
def test_steps_replayed_beside_each_other():
    """Graphs of whole steps of several states, replayed on streams of their own, and beside calls outside them."""
    states = [_step(s) for s in (3, 4, 5)]
    want = [_run(*s) for s in states]
    graphs, outs = [], []
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([_run(*s) for _ in range(3)])
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(4):
        for out in outs:
            for y in out:
                for t in y:
                    t.zero_()
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for out, ref in zip(outs, want):
            for y in out:
                assert all(torch.equal(a, b) for a, b in zip(y, ref))


def _program(text):
    r = subprocess.run([sys.executable, "-c", text], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_first_calls_may_be_captured():
    """Nothing that a first call sets up keeps it from being captured."""
    _program("""
import torch
from tests.test_gpu_decode_step import _run, _step
args = _step()
leaves = [args[2].clone().requires_grad_(), args[9].clone().requires_grad_()]
def step():
    from bitween_b200 import token_log_probs
    r = token_log_probs(leaves[1], args[10], entropy=True, top=2)
    y = args[0].rotate(args[6], leaves[0])
    return _run(*args) + [*torch.autograd.grad((y, r.log_probs, r.entropy), leaves, (torch.ones_like(y), torch.ones_like(r.log_probs), torch.ones_like(r.entropy)))]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
want = step()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("done")
""")


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_a_captured_backward_beside_a_living_graph_of_the_same_leaves(native):
    """Refused while the graph recorded on the default stream lives (on the Python path always); captured once it is gone."""
    _program(f"""
import torch
from bitween_b200 import RotaryPositions, token_log_probs
from bitween_b200.kernels import _lib
native = {native}
if not native:
    _lib._operators = _lib._NoOperators
rotary = RotaryPositions(64, 50)
q = torch.randn(9, 2, 64, device="cuda").half().requires_grad_()
x = torch.randn(9, 100, device="cuda").requires_grad_()
at = torch.arange(9, device="cuda")
calls = [(lambda: rotary.rotate(at, q), q), (lambda: token_log_probs(x, at).log_probs, x)]
for call, leaf in calls:
    living = call()
    grad = torch.ones_like(living)
    want = torch.autograd.grad(call(), leaf, grad)[0]
    torch.cuda.synchronize()
    refused = False
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
        try:
            torch.autograd.grad(y, leaf, grad)
        except RuntimeError as e:
            refused = "cannot be captured" in str(e)
    assert refused
    assert torch.equal(torch.autograd.grad(living, leaf, grad)[0], want)
    del living, y
    if native:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(call(), leaf, grad)[0]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
print("done")
""")
