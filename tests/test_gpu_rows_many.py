"""Sorts of more slots than 512 blocks of 1024 hold."""
import pytest
import torch

from fastmlx_amd import FmxqError, ops
from gpu_util import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,k,E,D", [(65536, 8, 64, 8), (65537, 8, 2048, 3), (600001, 3, 300, 8),
                                     (300000, 17, 7, 1)])
@pytest.mark.parametrize("bad", [False, True])
def test_sort_of_many_slots(gpu, T, k, E, D, bad):
    announce(f"sort {T}x{k} over {E}, bad ids {bad}")
    gen = torch.Generator().manual_seed(T)
    inds = torch.randint(0, E, (T, k), generator=gen).int().to(gpu)
    x = torch.randn(T, D, generator=gen).bfloat16().to(gpu)
    if bad:
        inds[5, 0], inds[T // 2, k - 1], inds[T - 1, 1] = E, -1, 2**31 - 1
    xs, order, pos, offsets = ops.moe_sort(x, inds, E)
    flat = inds.flatten().long()
    flat = torch.where((flat < 0) | (flat >= E), torch.full_like(flat, E), flat)
    want = torch.argsort(flat, stable=True)
    assert torch.equal(order.long(), want)
    assert torch.equal(pos.flatten().long()[want], torch.arange(T * k, device=gpu))
    count = torch.bincount(flat, minlength=E + 1)[:E]
    assert torch.equal(offsets.long(), torch.cat([count.new_zeros(1), count.cumsum(0)]))
    n = T * k - 3 * bad
    assert torch.equal(xs[:n], x[want[:n] // k]) and not xs[n:].any()
    if bad:
        with pytest.raises(FmxqError, match="INDEX"):
            ops.device_error()
    ops.device_error()
