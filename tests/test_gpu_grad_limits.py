"""Sizes at the ends of what the training operators take: widths, vocabularies and rows whose
launches or offsets are at their limits."""
import pytest
import torch

import grad_ref as ref
from fastmlx_amd import ops
from gpu_util import announce

pytestmark = pytest.mark.gpu


def test_quantized_matmul_grad_wider_than_a_panel(gpu):
    M, N, K = 1025, 16, 4180000
    announce(f"grad {M}x{N}x{K}")
    gen = torch.Generator().manual_seed(1)
    w = ref.quant(gen, (N,), K, 4, 32, gpu)
    dy = torch.randn(M, N, generator=gen).bfloat16().to(gpu)
    dx = ops.quantized_matmul_grad(dy, *w, 32, 4)
    W = ref.values(*w, 4, 32)
    for a in (0, 2 ** 21 - 500, K - 1000):
        ref.check(dx[:, a:a + 1000], *ref.product(dy, W[:, a:a + 1000]), f"columns from {a}")


def sampled(gpu, h, w, y, rows, group, got, grad):
    """Losses (and dh) of some rows against 64 bits."""
    W = ref.values(*w, 4, group)
    h, y = h[rows], y[rows].long()
    one = torch.ones(len(rows), device=gpu)
    (loss, el), (lse, es), (dh, ed) = ref.head(h, W, y[:, None], one.double()[:, None], one > 0, 1.0, one)
    ref.check(got[0][rows], loss, el, "loss")
    ref.check(got[1][rows], lse, es, "lse")
    if grad:
        ref.check(got[2][rows], dh, ed, "dh")


def test_cross_entropy_over_millions_of_tokens(gpu):
    """e's rows for one product would pass its 32-bit offsets: two pieces."""
    M, V, K = 20, 4300000, 512
    announce(f"ce {M}x{V}x{K}")
    gen = torch.Generator(device=gpu).manual_seed(2)
    w = (torch.randint(-2**31, 2**31, (V, K // 8), dtype=torch.int32, device=gpu, generator=gen),
         torch.empty(V, K // 64, device=gpu).uniform_(0.002, 0.02, generator=gen).bfloat16())
    w = (*w, -8 * w[1])
    h = torch.randn(M, K, device=gpu, generator=gen).bfloat16()
    y = torch.randint(0, V, (M,), device=gpu, generator=gen).int()
    y[0], y[1] = 0, V - 1
    got = ops.head_cross_entropy(h, *w, y, grad=True)
    sampled(gpu, h, w, y, torch.arange(M, device=gpu), 64, got, True)
    ops.device_error()


def test_cross_entropy_of_millions_of_rows(gpu):
    """More tiles than a launch has blocks: the vocabulary in two pieces."""
    M, V, K = 1 << 22, 131400, 32
    announce(f"ce {M}x{V}x{K}")
    gen = torch.Generator(device=gpu).manual_seed(3)
    w = (torch.randint(-2**31, 2**31, (V, K // 8), dtype=torch.int32, device=gpu, generator=gen),
         torch.empty(V, K // 32, device=gpu).uniform_(0.002, 0.02, generator=gen).bfloat16())
    w = (*w, -8 * w[1])
    h = torch.randn(M, K, device=gpu, generator=gen).bfloat16()
    y = torch.randint(0, V, (M,), device=gpu, generator=gen).int()
    rows = torch.tensor([0, 1, 255, 256, M // 2, M - 1, M - 2, M - 257], device=gpu)
    y[rows] = torch.tensor([0, V - 1, V - 300, 65792, 65700, 65536, 3, V // 2], device=gpu).int()
    got = ops.head_cross_entropy(h, *w, y, group_size=32)
    sampled(gpu, h, w, y, rows, 32, got, False)
    assert torch.isfinite(got[0]).all() and (got[0] >= 0).all()
    ops.device_error()
