"""Input gradients over weights whose dequantized panel is walked in pieces."""
import pytest
import torch

import grad_ref as ref
from fastmlx_amd import ops
from gpu_util import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K,bits,group", [
    (1025, 280000, 1024, 4, 64), (1030, 262147, 1056, 8, 32), (2000, 34001, 8192, 4, 128),
    (1026, 1100007, 512, 4, 64)])
def test_quantized_matmul_grad_in_pieces(gpu, M, N, K, bits, group):
    """More than 512 MB of bf16 weights: two pieces or three, the last one shorter, its rows cut inside
    a step where N is odd.  The memory is filled with NaN before, so that sums that were added to what
    the workspace held would show."""
    announce(f"grad in pieces {M}x{N}x{K} {bits} bits, groups of {group}")
    assert N * K * 2 > 512 << 20
    gen = torch.Generator().manual_seed(M)
    w = ref.quant(gen, (N,), K, bits, group, gpu)
    dy = torch.randn(M, N, generator=gen).bfloat16().to(gpu)
    y, e = None, None
    for a in range(0, N, 40000):  # in parts, for the 64-bit copies' memory
        W = ref.values(*(t[a:a + 40000] for t in w), bits, group)
        d = dy[:, a:a + 40000].double()
        part, size = d @ W, d.abs() @ W.abs()
        y, e = (part, size) if y is None else (y + part, e + size)
    # A sum of N products in 32 bits, and the results of the pieces and parts.
    e = (N + 64) * ref.U32 * e
    junk = torch.full((1 << 30,), 0xFF, dtype=torch.uint8, device=gpu)
    torch.cuda.synchronize()
    del junk
    dx = ops.quantized_matmul_grad(dy, *w, group, bits)
    ref.check(dx, y, e + ref.HALF[torch.bfloat16] * (y.abs() + e) + ref.TINY, "dx")
    # Rows do not depend on the other rows' number of tiles or parts by more than their sums' errors.
    one = ops.quantized_matmul_grad(dy[:7].contiguous(), *w, group, bits)
    ref.check(one, y[:7], (e + ref.HALF[torch.bfloat16] * (y.abs() + e) + ref.TINY)[:7], "seven rows")


@pytest.mark.parametrize("M,N,K", [(3, 16, 64), (40, 512, 256), (300, 4096, 128), (1100, 72, 128)])
@pytest.mark.parametrize("off", [1, 4, 7])
def test_rows_at_any_address(gpu, M, N, K, off):
    """Rows that begin between 16-byte addresses are moved to a workspace, and all the results are
    those of rows that do not."""
    announce(f"rows {off} values further, {M}x{N}x{K}")
    gen = torch.Generator().manual_seed(M)
    w = ref.quant(gen, (N,), K, 4, 64, gpu)
    dy = torch.randn(M, N, generator=gen).bfloat16().to(gpu)
    odd = torch.empty(M * N + off, dtype=torch.bfloat16, device=gpu)[off:].view(M, N).copy_(dy)
    two = tuple(torch.stack([t, t]) for t in w)
    ends = torch.tensor([0, M // 3, M], dtype=torch.int32, device=gpu)
    for path in (ops._fast, None):
        ops_fast, ops._fast = ops._fast, path
        try:
            assert torch.equal(ops.quantized_matmul_grad(odd, *w), ops.quantized_matmul_grad(dy, *w))
            assert torch.equal(ops.gather_qmm_grad(odd, *two, ends), ops.gather_qmm_grad(dy, *two, ends))
        finally:
            ops._fast = ops_fast
    ops.device_error()
