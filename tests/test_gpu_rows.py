"""Token rows sorted by expert and back, with gradients, on the GPU."""
import pytest
import torch

import grad_ref as ref
from fastmlx_amd import FmxqError, ops
from gpu_util import announce

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1, 1, 8), (1, 8, 256, 64), (16, 10, 512, 2048), (100, 3, 7, 100), (333, 6, 64, 1000),
          (1024, 1, 2, 16), (257, 4, 2048, 24), (700, 8, 5, 33), (3000, 8, 128, 256),
          (20000, 10, 300, 8), (40, 20, 64, 72), (90, 16, 30, 40), (128, 8, 2048, 1), (129, 8, 3, 520)]


def case(gpu, T, k, E, D, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed + T * k + E)
    x = torch.randn(T, D, generator=gen).bfloat16().to(gpu)
    inds = torch.randint(0, E, (T, k), generator=gen).int().to(gpu)
    w = torch.rand(T, k, generator=gen).to(dtype).to(gpu)
    y = torch.randn(T * k, D, generator=gen).bfloat16().to(gpu)
    dout = torch.randn(T, D, generator=gen).bfloat16().to(gpu)
    return x, inds, w, y, dout


@pytest.mark.parametrize("T,k,E,D", SHAPES)
def test_sort(gpu, T, k, E, D):
    announce(f"sort {T}x{k} over {E}, {D} wide")
    x, inds, _, y, _ = case(gpu, T, k, E, D, torch.float32)
    xs, order, pos, offsets = ops.moe_sort(x, inds, E)
    flat = inds.flatten().long()
    want = torch.argsort(flat, stable=True)
    assert torch.equal(order.long(), want)
    assert torch.equal(pos.flatten().long()[want], torch.arange(T * k, device=gpu))
    count = torch.bincount(flat, minlength=E)
    assert torch.equal(offsets.long(), torch.cat([count.new_zeros(1), count.cumsum(0)]))
    assert torch.equal(xs, x[want // k])
    dx = ops.moe_sort_grad(y, pos)
    v = y.double()[pos.long()]
    e = (k + 2) * ref.U32 * v.abs().sum(1)
    ref.check(dx, v.sum(1), e + ref.HALF[torch.bfloat16] * (v.sum(1).abs() + e), "dx")
    ops.device_error()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,k,E,D", SHAPES)
def test_unsort_and_gradients(gpu, T, k, E, D, dtype):
    announce(f"unsort {T}x{k} over {E}, {D} wide")
    x, inds, w, y, dout = case(gpu, T, k, E, D, dtype)
    pos = ops.moe_sort(x, inds, E)[2]
    half = ref.HALF[torch.bfloat16]
    v = y.double()[pos.long()]
    terms = v * w.double()[..., None]
    e = (k + 2) * ref.U32 * terms.abs().sum(1)
    ref.check(ops.moe_unsort(y, pos, w), terms.sum(1), e + half * (terms.sum(1).abs() + e), "out")
    dy, dw = ops.moe_unsort_grad(dout, y, pos, w)
    assert dw.dtype == dtype
    full = (w.double()[..., None] * dout.double()[:, None, :])
    # fp32 product, then bf16: two roundings.
    ref.check(dy[pos.long()], full, (half + 2 * ref.U32) * full.abs() + ref.TINY, "dy")
    dots = v * dout.double()[:, None, :]
    e = (D + 2) * ref.U32 * dots.abs().sum(-1)
    ref.check(dw, dots.sum(-1), e + ref.HALF[dtype] * (dots.sum(-1).abs() + e), "dweights")
    ops.device_error()


def test_sums_of_rows_larger_than_the_cache(gpu):
    T, k, E, D = 4200, 8, 16, 4096
    announce(f"sums {T}x{k}, {D} wide")
    x, inds, w, y, _ = case(gpu, T, k, E, D, torch.bfloat16)
    pos = ops.moe_sort(x, inds, E)[2]
    half = ref.HALF[torch.bfloat16]
    for got, weights in ((ops.moe_unsort(y, pos, w), w.double()),
                         (ops.moe_sort_grad(y, pos), torch.ones_like(w).double())):
        for t in range(0, T, 700):  # in parts, for the 64-bit copies' memory
            terms = y[pos[t:t + 700].long()].double() * weights[t:t + 700, :, None]
            e = (k + 2) * ref.U32 * terms.abs().sum(1)
            ref.check(got[t:t + 700], terms.sum(1), e + half * (terms.sum(1).abs() + e), "sums")
    ops.device_error()


def test_empty(gpu):
    announce("no tokens")
    x = torch.empty(0, 16, dtype=torch.bfloat16, device=gpu)
    inds = torch.empty(0, 4, dtype=torch.int32, device=gpu)
    xs, order, pos, offsets = ops.moe_sort(x, inds, 6)
    assert xs.shape == (0, 16) and order.shape == (0,) and pos.shape == (0, 4)
    assert offsets.tolist() == [0] * 7
    w = torch.empty(0, 4, device=gpu)
    assert ops.moe_unsort(xs, pos, w).shape == (0, 16)
    assert ops.moe_sort_grad(xs, pos).shape == (0, 16)
    dy, dw = ops.moe_unsort_grad(x, xs, pos, w)
    assert dy.shape == (0, 16) and dw.shape == (0, 4)


@pytest.mark.parametrize("T", [9, 2000])
def test_ids_out_of_range(gpu, T):
    """Bad ids sort last in slot order, with zero rows, and are reported."""
    announce(f"bad ids, {T} tokens")
    x, inds, w, y, dout = case(gpu, T, 3, 4, 40, torch.float32)
    inds[1, 2], inds[5, 0], inds[T - 1, 1] = 4, -1, 2**31 - 1
    xs, order, pos, offsets = ops.moe_sort(x, inds, 4)
    with pytest.raises(FmxqError, match="INDEX"):
        ops.device_error()
    assert int(offsets[4]) == 3 * T - 3
    assert order[-3:].tolist() == [5, 15, 3 * (T - 1) + 1]
    assert not xs[-3:].any()
    assert torch.equal(xs[:-3], x[order[:-3].long() // 3])
    ops.device_error()


def test_positions_out_of_range(gpu):
    announce("bad positions")
    x, inds, w, y, dout = case(gpu, 6, 2, 3, 16, torch.float32)
    pos = ops.moe_sort(x, inds, 3)[2]
    kept = pos.clone()
    pos[2, 1] = 12
    pos[4, 0] = -1
    out = ops.moe_unsort(y, pos, w)
    with pytest.raises(FmxqError, match="INDEX"):
        ops.device_error()
    w2 = w.clone()
    w2[2, 1] = w2[4, 0] = 0
    assert torch.equal(out, ops.moe_unsort(y, kept, w2))
    _, dw = ops.moe_unsort_grad(dout, y, pos, w)
    assert dw[2, 1] == 0 and dw[4, 0] == 0
    with pytest.raises(FmxqError, match="INDEX"):
        ops.device_error()


def test_a_training_step_of_an_expert_layer_and_the_head(gpu):
    """Router weights, sorted experts, the way back and the head's loss, forward and backward,
    against 64-bit autograd of the same formulas."""
    announce("step")
    gen = torch.Generator().manual_seed(2)
    T, k, E, D, I, V = 60, 2, 6, 128, 256, 400
    q = [ref.quant(gen, (E, n), d, 4, 64, gpu) for n, d in ((I, D), (I, D), (D, I))]
    head = ref.quant(gen, (V,), D, 4, 64, gpu)
    x = torch.randn(T, D, generator=gen).bfloat16().to(gpu)
    y = torch.randint(0, V, (T,), generator=gen).int().to(gpu)
    inds, weights = ops.route_softmax_topk(torch.randn(T, E, generator=gen).bfloat16().to(gpu), k,
                                           weights_dtype=torch.float32)
    xs, order, pos, offsets = ops.moe_sort(x, inds, E)
    ids = inds.flatten()[order.long()].contiguous()

    def product(a, m):
        return ops.gather_qmm(a[:, None, :].contiguous(), *m, ids, sorted_indices=True)[:, 0]

    gate, up = product(xs, q[0]).float(), product(xs, q[1]).float()
    s = torch.sigmoid(gate)
    hmid = (gate * s * up).bfloat16()
    yr = product(hmid, q[2]).contiguous()
    out = ops.moe_unsort(yr, pos, weights)
    h = (x.float() + out.float()).bfloat16()
    mean = torch.full((T,), 1.0 / T, device=gpu)
    loss, _, dh = ops.head_cross_entropy(h, *head, y, grad=True, grad_loss=mean)
    dy, dweights = ops.moe_unsort_grad(dh, yr, pos, weights)
    dmid = ops.gather_qmm_grad(dy, *q[2], offsets).float()
    dgate = (dmid * up * (s + gate * s * (1 - s))).bfloat16()
    dup = (dmid * gate * s).bfloat16()
    dxs = ops.gather_qmm_grad(dgate, *q[0], offsets).float()
    dxs = (dxs + ops.gather_qmm_grad(dup, *q[1], offsets).float()).bfloat16()
    dx = ops.moe_sort_grad(dxs, pos).float() + dh.float()
    ops.device_error()

    W = [ref.values(*m, 4, 64) for m in q]
    xr = x.double().requires_grad_()
    wr = weights.double().requires_grad_()
    e = inds.long()
    g = torch.einsum("td,tjid->tji", xr, W[0][e])
    u = torch.einsum("td,tjid->tji", xr, W[1][e])
    z = torch.einsum("tji,tjdi->tjd", g * torch.sigmoid(g) * u, W[2][e])
    hr = xr + (wr[..., None] * z).sum(1)
    logits = hr @ ref.values(*head, 4, 64).T
    lr = torch.nn.functional.cross_entropy(logits, y.long(), reduction="none")
    lr.mean().backward()
    # The chain rounds to bf16 ten times (gate, up, their product, down, out, h, dh, dy, dgate /
    # dup, dxs, dx): each off by at most 2^-8 of its size, taken as a norm; the products' sums
    # and the softmax pass relative errors on with a factor near 1 at these sizes.
    tol = 10 * 2.0 ** -8

    def near(a, b):
        return float((a.double() - b).norm() / b.norm())

    assert near(loss, lr.detach()) < tol
    assert near(dx, xr.grad) < tol
    assert near(dweights, wr.grad) < tol
