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


@pytest.mark.parametrize("M,V", [(12, 900), (150, 30000), (1100, 12000)])
def test_gradients_of_logits_beyond_the_exponents_range(gpu, M, V):
    """Logits of 1e9 and more, the largest of a row further from the others than any error of
    theirs: one token takes everything, and dh is the difference of two rows of the weights."""
    announce(f"gradients of huge logits {M}x{V}")
    gen = torch.Generator().manual_seed(M)
    K = 256
    w = ref.quant(gen, (V,), K, 4, 64, gpu)
    W = ref.values(*w, 4, 64)
    h = torch.randn(M, K, generator=gen).to(gpu)
    h = (h * torch.logspace(8, 24, M, device=gpu)[:, None]).bfloat16()
    logits = h.double() @ W.T
    (first, second), ids = (lambda t: (t.values.T, t.indices))(logits.topk(2, -1))
    error = (K + 16) * ref.U32 * (h.double().abs() @ W.abs().T).amax(-1)
    apart = first - second > 4 * error
    assert apart.double().mean() > 0.9
    y = torch.randint(0, V, (M,), generator=gen).to(gpu)
    y[::3] = ids[::3, 0]          # some rows want the token that they take
    g = (torch.rand(M, generator=gen) + 0.5).to(gpu)
    dh = g.double()[:, None] * (W[ids[:, 0]] - W[y])
    # The taken token's share is a power of two in bf16, half a step off at most; the wanted one's
    # and the sums are fp32.
    size = g.double()[:, None] * (W[ids[:, 0]].abs() + W[y].abs())
    e = (ref.HALF[torch.bfloat16] + 64 * ref.U32) * size
    e = e + ref.HALF[torch.bfloat16] * (dh.abs() + e)
    got = ops.head_cross_entropy(h, *w, y.int(), grad=True, grad_loss=g)
    ref.check(got[2][apart], dh[apart], e[apart], "dh")
    same = apart & (y == ids[:, 0])
    assert same.any() and not got[2][same].any() and not got[0][same].any()
    # One entry of a teacher is the same, at any temperature.
    got = ops.head_distill((h * 0 + 1).bfloat16(), *w, y.int()[:, None].contiguous(),
                           torch.zeros(M, 1, device=gpu), temperature=1e-10, grad=True)
    top = W.sum(-1).topk(2)
    assert top.values[0] - top.values[1] > 4 * (K + 16) * ref.U32 * W.abs().sum(-1).max()
    at = int(top.indices[0])
    dh = 1e-10 * (W[at] - W[y])
    size = 1e-10 * (W[at].abs() + W[y].abs())
    e = (ref.HALF[torch.bfloat16] + 64 * ref.U32) * size
    ref.check(got[2], dh, e + ref.HALF[torch.bfloat16] * (dh.abs() + e), "dh at 1e-10")
