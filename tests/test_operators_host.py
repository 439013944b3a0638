"""The checks of the cache's and the adapters' arguments, which need no GPU."""
import pytest
import torch

from bitween_b200 import AdaptedLinear, QuantizedKVCache, QuantizedLinear, adapter_matmul
from bitween_b200.kernels import _lib

P = 1 << 20      # an aligned address that no call here reaches


def test_cache_entry_points_check_their_arguments():
    L = _lib.lib()

    def append(dtype=1, tokens=4, heads=2, dim=64, bits=4, pages=3, page=16, k=P, slots=P, codes=P):
        return L.bw_kv_append(k, P, dtype, tokens, 128, 64, 128, 64, slots, heads, dim, bits, pages, page, codes, P, P, None)

    assert append(bits=3) == 1
    assert append(dim=60) == 3 and append(dim=264) == 3 and append(dim=0) == 3 and append(heads=0) == 3 and append(page=0) == 3 and append(pages=-1) == 3
    assert append(tokens=-1) == 3 and append(tokens=1 << 40) == 3
    assert append(dtype=3) == 4
    assert append(k=P + 1) == 5 and append(codes=P + 4) == 5 and append(slots=P + 4) == 5
    assert append(k=None) == 6 and append(slots=None) == 6 and append(codes=None) == 6
    assert append(tokens=0) == 0 and append(pages=0, codes=None) == 0

    def read(dtype=1, tokens=4, k=P, bits=8, slots=P):
        return L.bw_kv_read(P, P, P, 2, 64, bits, 3, 16, slots, tokens, k, P, dtype, None)

    assert read(bits=5) == 1 and read(dtype=9) == 4 and read(tokens=-2) == 3 and read(k=P + 2) == 5 and read(slots=None) == 6 and read(tokens=0) == 0

    def attend(dtype=1, batch=2, heads=4, kv_heads=2, dim=64, table=P, stride=4, wide=4, q=P, lengths=P, ws=P, size=1 << 40):
        return L.bw_kv_attend(q, dtype, batch, heads, heads * dim, dim, P, P, P, 4, 3, 16, kv_heads, dim, table, stride, wide, lengths, 0.1, P, ws, size, None)

    assert attend(dtype=0) == 4 and attend(heads=3) == 3 and attend(batch=-1) == 3 and attend(wide=1 << 31) == 3 and attend(stride=-1) == 3
    assert attend(q=None) == 6 and attend(table=None) == 6 and attend(lengths=None) == 6
    assert attend(q=P + 1) == 5 and attend(table=P + 2) == 5
    assert attend(batch=0) == 0
    need = L.bw_kv_attend_workspace_bytes(2, 4, 2, 64, 16, 1 << 20)
    if need:
        assert attend(wide=1 << 20, ws=None) == 7 and attend(wide=1 << 20, size=need - 1) == 7 and attend(wide=1 << 20, ws=P + 8) == 5
    assert L.bw_kv_attend_workspace_bytes(0, 4, 2, 64, 16, 4) == 0 and L.bw_kv_attend_workspace_bytes(2, 4, 0, 64, 16, 4) == 0


def test_adapter_entry_points_check_their_arguments():
    L = _lib.lib()

    def forward(dtype=1, M=4, N=64, K=64, n=2, r=8, x=P, index=P, hidden=P, size=1 << 40, out=P):
        return L.bw_adapter_forward(x, dtype, M, N, K, P, P, n, r, index, None, None, out, hidden, size, None)

    assert forward(dtype=0) == 4 and forward(dtype=3) == 4
    assert forward(M=-1) == 3 and forward(n=0) == 3 and forward(r=0) == 3 and forward(r=257) == 3 and forward(K=0) == 3 and forward(N=1 << 25) == 3
    assert forward(x=None) == 6 and forward(index=None) == 6 and forward(out=None) == 6
    assert forward(x=P + 1) == 5 and forward(index=P + 2) == 5 and forward(hidden=P + 4) == 5
    assert forward(hidden=None) == 7 and forward(size=L.bw_adapter_hidden_bytes(4, 8) - 1) == 7
    assert forward(M=0) == 0

    def backward(M=4, x=P, hidden=P, size=1 << 40, ws=P, wsize=1 << 40, dtype=2):
        return L.bw_adapter_backward(P, dtype, x, M, 64, 64, P, P, 2, 8, P, None, hidden, size, P, P, P, ws, wsize, None)

    assert backward(dtype=0) == 4 and backward(M=-1) == 3 and backward(x=None) == 6 and backward(x=P + 1) == 5 and backward(ws=P + 4) == 5
    assert backward(hidden=None) == 7 and backward(size=8) == 7 and backward(ws=None) == 7 and backward(wsize=8) == 7
    assert L.bw_adapter_hidden_bytes(0, 8) == 0 and L.bw_adapter_hidden_bytes(4, 8) == 4 * 8 * 4 + 16


def test_cache_refusals():
    for args in ((4, 16, 2, 60, 4), (4, 16, 2, 264, 8), (4, 0, 2, 64, 8), (4, 16, 0, 64, 8), (-1, 16, 2, 64, 8), (4, 16, 2, 64, 3)):
        with pytest.raises(ValueError):
            QuantizedKVCache(*args, device="cpu")
    cache = QuantizedKVCache(4, 16, 2, 64, bits=4, device="cpu")
    assert cache.k_codes.shape == (4, 2, 16, 8) and cache.params.shape == (4, 2, 16, 4) and "head_dim=64" in repr(cache)
    same = QuantizedKVCache.from_tensors(cache.k_codes, cache.v_codes, cache.params, 4)
    assert (same.head_dim, same.num_pages, same.page_size, same.num_kv_heads) == (64, 4, 16, 2) and same.k_codes is cache.k_codes
    k, v, p = cache.k_codes, cache.v_codes, cache.params
    for bad in ((k, v, p, 5), (k.long(), v, p, 4), (k, v[:3], p, 4), (k, v, p.float(), 4), (k, v, p[..., :2], 4), (k[0], v[0], p[0], 4),
                (k[:, :, ::2], v[:, :, ::2], p[:, :, ::2].contiguous(), 4), (k.view(4, 2, 8, 16).repeat(1, 1, 1, 4), v.view(4, 2, 8, 16).repeat(1, 1, 1, 4), p[:, :, :8].contiguous(), 4)):
        with pytest.raises(ValueError):
            QuantizedKVCache.from_tensors(*bad)
    slots, x = torch.arange(3), torch.zeros(3, 2, 64)
    with pytest.raises(RuntimeError):
        cache.append(x, x, slots)                      # no CPU path
    with pytest.raises(RuntimeError):
        cache.read(slots)
    with pytest.raises(TypeError):
        cache.read(slots, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        cache.attend(x.half(), torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32))


def test_adapter_refusals():
    x = torch.zeros(3, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError):
        adapter_matmul(x, torch.zeros(1, 8, 64).half(), torch.zeros(1, 8, 32).half(), torch.zeros(3, dtype=torch.int32))
    layer = QuantizedLinear(64, 32, bits=4, group_size=32)
    adapted = AdaptedLinear(layer, 2, 8)
    assert adapted.down.shape == (2, 8, 64) and adapted.up.shape == (2, 8, 32) and not adapted.up.any()
    for bad in ((torch.nn.Linear(4, 4), 1, 8), (layer, 0, 8), (layer, 1, 0), (layer, 1, 257)):
        with pytest.raises((TypeError, ValueError)):
            AdaptedLinear(*bad)
    with pytest.raises(TypeError):
        AdaptedLinear(layer, 1, 8, dtype=torch.float32)


@pytest.mark.gpu
def test_refusals_of_tensors_on_the_gpu():
    dev = "cuda"
    cache = QuantizedKVCache(4, 16, 2, 64, bits=4, device=dev)
    slots, x = torch.arange(3, device=dev), torch.zeros(3, 2, 64, device=dev).half()
    i32 = {"dtype": torch.int32, "device": dev}
    for error, call in (
            (TypeError, lambda: cache.append(x, x, slots.int())), (RuntimeError, lambda: cache.append(x, x, slots.cpu())),
            (ValueError, lambda: cache.append(x[:2], x, slots)), (ValueError, lambda: cache.append(x, x[..., :32], slots)),
            (TypeError, lambda: cache.append(x, x.float(), slots)), (TypeError, lambda: cache.append(x.double(), x.double(), slots)),
            (RuntimeError, lambda: cache.append(x.cpu(), x.cpu(), slots)), (TypeError, lambda: cache.read(slots.int())),
            (TypeError, lambda: cache.attend(x.float(), torch.zeros(3, 1, **i32), torch.ones(3, **i32))),
            (ValueError, lambda: cache.attend(x[:, :1], torch.zeros(3, 1, **i32), torch.ones(3, **i32))),
            (ValueError, lambda: cache.attend(x[..., :32], torch.zeros(3, 1, **i32), torch.ones(3, **i32))),
            (TypeError, lambda: cache.attend(x, torch.zeros(3, 1, device=dev).long(), torch.ones(3, **i32))),
            (ValueError, lambda: cache.attend(x, torch.zeros(2, 1, **i32), torch.ones(3, **i32))),
            (ValueError, lambda: cache.attend(x, torch.zeros(3, 1, **i32), torch.ones(2, **i32))),
            (RuntimeError, lambda: cache.attend(x, torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, **i32)))):
        with pytest.raises(error):
            call()
    x, down, up, index = torch.zeros(3, 64, device=dev).half(), torch.zeros(2, 8, 64, device=dev).half(), torch.zeros(2, 8, 32, device=dev).half(), torch.zeros(3, **i32)
    base = torch.zeros(3, 32, device=dev).half()
    f = torch.ones(2, device=dev)
    for error, call in (
            (TypeError, lambda: adapter_matmul(x.float(), down, up, index)), (TypeError, lambda: adapter_matmul(x, down.bfloat16(), up, index)),
            (ValueError, lambda: adapter_matmul(x[:, :32], down, up, index)), (ValueError, lambda: adapter_matmul(x, down, up[:1], index)),
            (TypeError, lambda: adapter_matmul(x, down, up, index.long())), (ValueError, lambda: adapter_matmul(x, down, up, index[:2])),
            (ValueError, lambda: adapter_matmul(x, down, up, index, base=base[:2])), (TypeError, lambda: adapter_matmul(x, down, up, index, base=base.float())),
            (ValueError, lambda: adapter_matmul(x, down, up, index, scaling=f[:1])), (ValueError, lambda: adapter_matmul(x, down, up, index, scaling=f.half())),
            (ValueError, lambda: adapter_matmul(x, down, up, index, scaling=f.clone().requires_grad_())),
            (RuntimeError, lambda: adapter_matmul(x, down, up, index.cpu())), (ValueError, lambda: adapter_matmul(x, down[:0], up[:0], index)),
            (ValueError, lambda: adapter_matmul(x, down.requires_grad_(), up, index, base=base, out=base)),
            (ValueError, lambda: adapter_matmul(x, down.detach(), up, index, out=base[:2]))):
        with pytest.raises(error):
            call()
