"""Attention over the quantised cache where its work is divided: the line of work over many sequences, clusters, and marks of bad pages in either."""
import pytest
import torch

from bitween_b200.kernels import _lib
from test_gpu_kv_cache import _attended, _check, _filled, _gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHARES, ONE_LAUNCH, GENERAL = "kv_attend_join_kernel", "kv_attend_kernel", "kv_attend_general_kernel"


def _mixed(batch, seed, longest):
    """Lengths of 0, of 1 and of thousands; whole runs of 32 empty ones."""
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(0, 5, (batch,), generator=g)
    long = torch.randint(1, longest + 1, (batch,), generator=g)
    lengths = torch.where(n == 0, 0, torch.where(n == 1, 1, long))
    if batch >= 64:
        lengths[:32] = 0
    if batch >= 96:
        lengths[64:96] = 0
    lengths[batch // 2] = longest
    return lengths.tolist()


@pytest.mark.parametrize("batch,heads,kv_heads,dim,bits,longest", [
    (33, 8, 2, 128, 4, 3000), (33, 8, 2, 128, 4, 6000), (64, 4, 1, 64, 8, 5000), (96, 8, 2, 128, 2, 2000), (97, 5, 1, 256, 4, 3000), (130, 20, 2, 64, 4, 1500), (33, 32, 8, 128, 4, 4000), (64, 1, 1, 64, 4, 40000)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_sequences_share_the_line_of_work(batch, heads, kv_heads, dim, bits, longest, dtype):
    lengths = _mixed(batch, batch + dim, longest)
    cache, table, n, slots = _filled(lengths, kv_heads, dim, bits, 16, 40)
    q = torch.randn(batch, heads, dim, generator=_gen(41), device=DEV).to(dtype)
    got = cache.attend(q, table, n)
    assert _lib.last_kernel() == (ONE_LAUNCH if (batch, longest) == (33, 3000) else SHARES)
    want, size = _attended(cache, q, slots, lengths, dim ** -0.5)
    _check(got, want, size)
    assert bool((got[n == 0] == 0).all())
    assert torch.equal(got, cache.attend(q, table, n))
    nothing = cache.attend(q, table, torch.zeros_like(n))
    assert bool((nothing == 0).all())


@pytest.mark.parametrize("lengths,kernel", [
    ([5000, 3000, 4999, 1, 6000, 2500], SHARES),            # parts of a sequence on many CTAs
    ([700, 900, 400, 1, 1000, 300], ONE_LAUNCH),            # clusters of several CTAs
    ([40, 60, 40, 1, 64, 30], ONE_LAUNCH),                  # of one
])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_bad_pages_and_lengths_wherever_a_sequence_is_divided(lengths, kernel, where):
    """A page outside the cache, a length beyond the table or below zero: NaN, NaN and zeros for that sequence alone, whichever part of it is concerned."""
    cache, table, n, slots = _filled(lengths, 2, 128, 4, 16, 50)
    q = torch.randn(6, 8, 128, generator=_gen(51), device=DEV).half()
    want, size = _attended(cache, q, slots, lengths, 128 ** -0.5)
    for b, page in ((0, cache.num_pages), (1, -1)):
        last = (lengths[b] - 1) // 16
        table[b, {"first": 0, "middle": last // 2, "last": last}[where]] = page
    table[3, 1:] = 2 ** 31 - 1                               # (one token: not reached)
    n[2], n[4] = -7, table.shape[1] * 16 + 1
    got = cache.attend(q, table, n)
    assert _lib.last_kernel() == kernel
    assert bool(got[[0, 1, 4]].isnan().all()) and bool((got[2] == 0).all())
    _check(got[[3, 5]], want[[3, 5]], size[[3, 5]])
    assert _lib.lib().bw_device_status() == 0


@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page,kernel", [
    ([40, 9, 0], 6, 3, 80, 16, GENERAL), ([100, 33], 4, 2, 128, 7, GENERAL), ([49], 12, 12, 64, 16, ONE_LAUNCH), ([257, 31], 32, 2, 256, 32, ONE_LAUNCH),
    ([20011], 4, 2, 128, 16, SHARES), ([5000], 5, 1, 64, 16, SHARES)])
def test_which_kernels_run(lengths, heads, kv_heads, dim, page, kernel):
    """The sizes by which the tests mean a form of the kernel reach it."""
    cache, table, n, _ = _filled(lengths, kv_heads, dim, 4, page, 60)
    cache.attend(torch.zeros(len(lengths), heads, dim, dtype=torch.float16, device=DEV), table, n)
    assert _lib.last_kernel() == kernel
