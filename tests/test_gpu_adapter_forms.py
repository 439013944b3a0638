"""Which of their kernels the adapters' passes take: the sizes by which the tests mean a form reach it."""
import pytest
import torch

from bitween_b200.kernels import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ran(M, K, N, n, r, dtype):
    """Names of the last kernel of a forward pass, of one for dx alone, for d_down alone and for d_up alone."""
    L = _lib.lib()
    x, dy, down, up = (torch.zeros(s, dtype=dtype, device=DEV) for s in ((M, K), (M, N), (n, r, K), (n, r, N)))
    index = torch.zeros(M, dtype=torch.int32, device=DEV)
    need = L.bw_adapter_hidden_bytes(M, r)
    hidden, ws = (torch.zeros(need, dtype=torch.uint8, device=DEV) for _ in range(2))
    y, dx, ddown, dup = (torch.ones_like(t) for t in (dy, x, down, up))
    code, stream, names = _lib.dtype_code(dtype), torch.cuda.current_stream().cuda_stream, []
    _lib.check(L.bw_adapter_forward(x.data_ptr(), code, M, N, K, down.data_ptr(), up.data_ptr(), n, r, index.data_ptr(), None, None, y.data_ptr(), hidden.data_ptr(), need, stream))
    names.append(_lib.last_kernel())
    for i, t in enumerate((dx, ddown, dup)):
        out = [t.data_ptr() if i == j else None for j in range(3)]
        _lib.check(L.bw_adapter_backward(dy.data_ptr(), code, x.data_ptr(), M, N, K, down.data_ptr(), up.data_ptr(), n, r, index.data_ptr(), None, hidden.data_ptr(), need, *out,
                                         ws.data_ptr(), need, stream))
        names.append(_lib.last_kernel())
    assert all(bool((t == 0).all()) for t in (y, dx, ddown, dup)) and L.bw_device_status() == 0
    return [s.removeprefix("adapter_").removesuffix("_kernel") for s in names]


@pytest.mark.parametrize("M,K,N,n,r,dtype,forms", [
    (64, 256, 256, 1, 128, torch.float16, ["expand_few", "expand_few", "outer", "outer"]),
    (130, 1088, 960, 5, 16, torch.float16, ["expand", "expand", "outer", "outer"]),
    (7, 100, 130, 3, 5, torch.float16, ["expand_general", "expand_general", "outer_general", "outer_general"]),
    (40, 4096, 96, 2, 1, torch.bfloat16, ["expand_general", "expand_general", "outer_general", "outer_general"]),
    (33, 8, 128, 2, 256, torch.bfloat16, ["expand_general", "expand_general", "outer_general", "outer_general"]),
    (512, 4096, 4096, 16, 64, torch.bfloat16, ["expand", "expand", "outer", "outer"]),
    (512, 4096, 14336, 1, 64, torch.bfloat16, ["expand_umma", "expand", "outer_umma", "outer_umma"]),
    (1024, 1024, 4096, 1, 32, torch.float16, ["expand", "expand", "outer", "outer_umma"]),
    (8192, 64, 1024, 1, 16, torch.bfloat16, ["expand", "expand", "outer", "outer"]),
    # sums over many tokens on tcgen05
    (512, 64, 264, 1, 64, torch.bfloat16, ["expand", "expand", "outer_umma", "outer_umma"]),
    (1023, 64, 2048, 2, 128, torch.bfloat16, ["expand", "expand", "outer_umma", "outer_umma"]),
    (2048, 64, 1000, 1, 32, torch.bfloat16, ["expand", "expand", "outer_umma", "outer_umma"]),
    (2049, 64, 136, 3, 24, torch.float16, ["expand", "expand", "outer_umma", "outer_umma"]),
    (17000, 64, 128, 2, 64, torch.float16, ["expand", "expand", "outer_umma", "outer_umma"]),
    # results of many tokens on tcgen05
    (1027, 64, 8200, 1, 64, torch.float16, ["expand_umma", "expand", "outer_umma", "outer_umma"]),
    (2050, 128, 12296, 3, 128, torch.bfloat16, ["expand_umma", "expand", "outer_umma", "outer_umma"]),
    (6300, 64, 4000, 5, 40, torch.float16, ["expand_umma", "expand", "outer_umma", "outer_umma"]),
    (24600, 64, 1032, 2, 48, torch.bfloat16, ["expand_umma", "expand", "outer_umma", "outer_umma"]),
])
def test_which_kernels_run(M, K, N, n, r, dtype, forms):
    assert _ran(M, K, N, n, r, dtype) == forms
