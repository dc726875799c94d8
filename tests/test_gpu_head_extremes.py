"""Teachers and temperatures at the ends of what a distillation takes."""
import pytest
import torch

import grad_ref as ref
from fastmlx_amd import ops
from gpu_util import announce

pytestmark = pytest.mark.gpu


def case(gpu, M=6, V=500, K=128, k=4, seed=1):
    gen = torch.Generator().manual_seed(seed)
    w = ref.quant(gen, (V,), K, 4, 64, gpu)
    h = torch.randn(M, K, generator=gen).bfloat16().to(gpu)
    ids = torch.stack([torch.randperm(V, generator=gen)[:k] for _ in range(M)]).int().to(gpu)
    return h, w, ids, gen


def check(h, w, ids, t, T=1.0):
    W = ref.values(*w, 4, 64)
    at, q, keep = ref.teacher_q(ids, t, W.shape[0], T)
    want = ref.head(h, W, at, q, keep, T, torch.ones(len(h), device=h.device))
    got = ops.head_distill(h, *w, ids, t, temperature=T, grad=True)
    only = ops.head_distill(h, *w, ids, t, temperature=T)
    for name, a, (r, e) in zip(("loss", "lse", "dh"), got, want):
        ref.check(a, r, e, name)
    for name, a, (r, e) in zip(("loss", "lse"), only, want):
        ref.check(a, r, e, name + " alone")
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_teacher_rows_of_the_types_lowest_value(gpu, dtype):
    """Finite logits, all alike: every entry has the same weight, and the row its loss."""
    announce(f"lowest teacher, {dtype}")
    h, w, ids, _ = case(gpu)
    low = torch.finfo(dtype).min
    t = torch.full(ids.shape, low, dtype=dtype, device=gpu)
    t[1, 2] = float("-inf")       # one of them absent in effect
    t[2] = float("-inf")          # no entry
    t[3, 0] = 5.0                 # the others far below
    ids[4, 1:] = -1               # one entry, the lowest
    t[5] = torch.finfo(dtype).max
    loss = check(h, w, ids, t)[0]
    assert loss[0] > 1 and loss[2] == 0
    check(h, w, ids, t, T=0.25)
    ops.device_error()


@pytest.mark.parametrize("T", [1e-25, 1e-15, 1e15])
def test_temperatures_whose_square_leaves_the_range(gpu, T):
    """T^2 = 1e-50 is no fp32 number, the loss (the divergence is near a logit / T) is one."""
    announce(f"temperature {T}")
    h, w, ids, gen = case(gpu)
    t = torch.randn(ids.shape, generator=gen).to(gpu)
    loss = check(h, w, ids, t, T)[0]
    assert (loss > 0).all()
