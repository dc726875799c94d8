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
