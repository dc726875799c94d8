"""Losses and gradients of rows that are sure of what they want, relative to their own size.

A cross entropy is log(1 + x) with x the sum of exp(l_v - l_y) over the other tokens: an error of
the logits by at most d moves log x by at most 2 d, so it moves the loss by no more than that part
of the loss itself, however small it is.  The bounds here say so (tests/grad_ref.py holds a loss to
the size of the logits instead).
"""
import pytest
import torch

import grad_ref as ref
from fastmlx_amd import ops
from gpu_util import announce

pytestmark = pytest.mark.gpu


def logit_error(h, W, T):
    """How far a logit / T may be off: an fp32 sum of K products, and eight roundings of its size
    (the scaling, its difference from a power of two's exponent, exp2 and log2)."""
    size = (h.double().abs() @ W.abs().T).amax(-1) / T
    return (h.shape[1] + 16) * ref.U32 * size


def sums_error(V):
    """Relative: fp32 sums over a tile's tokens and over tiles, and some roundings."""
    return (min(V, 2048) + 192) * ref.U32


def sure(gen, W, y, most):
    """Hidden states along W_y, so far that the wanted logit leads by 0 to `most`."""
    at = torch.arange(len(y), device=W.device)
    near = W[y] @ W.T
    own = near[at, y]
    near[at, y] = -torch.inf
    lead = torch.linspace(0, most, len(y), dtype=torch.float64, device=W.device)
    return (W[y] * (lead / (own - near.amax(-1)))[:, None]).bfloat16()


@pytest.mark.parametrize("M,V,K,bits,group", [
    (24, 900, 512, 4, 64), (1, 3000, 256, 4, 64), (40, 5000, 256, 8, 64), (64, 2000, 320, 4, 32),
    (200, 1200, 256, 4, 64),                           # the kernel for few rows
    (100, 40000, 256, 4, 128), (300, 20000, 512, 4, 32), (200, 30001, 192, 8, 64),   # tiles
    (1100, 24001, 320, 4, 64), (1900, 14000, 256, 8, 128)])                          # panels
def test_cross_entropy_of_sure_rows(gpu, M, V, K, bits, group):
    announce(f"sure rows {M}x{V}x{K} {bits} bits, groups of {group}")
    gen = torch.Generator().manual_seed(M + V)
    w = ref.quant(gen, (V,), K, bits, group, gpu)
    W = ref.values(*w, bits, group)
    y = torch.randint(0, V, (M,), generator=gen).to(gpu)
    h = sure(gen, W, y, 45.0) if M > 1 else sure(gen, W, y.repeat(2), 30.0)[1:]
    g = (torch.rand(M, generator=gen) + 0.1).to(gpu)

    logits = h.double() @ W.T
    own = logits.gather(1, y[:, None])[:, 0]
    logits.scatter_(1, y[:, None], -torch.inf)
    x = torch.logsumexp(logits, -1) - own  # log of the others' share over the wanted one's
    loss = torch.logaddexp(x, torch.zeros_like(x))
    assert loss.min() < 1e-10 and (M == 1 or loss.max() > 1)
    rel = torch.expm1(2 * logit_error(h, W, 1.0)) + sums_error(V)
    assert rel.median() < 0.01  # the bound says something
    eloss = loss * rel + ref.TINY
    lse = own + loss
    # The gradient: what the others leave, both times.
    rest = torch.sigmoid(x)
    p = (logits - lse[:, None]).exp()
    dh = g.double()[:, None] * (p @ W - rest[:, None] * W[y])
    others = g.double()[:, None] * (p @ W.abs())
    edh = others * (ref.HALF[torch.bfloat16] + 2 * rel[:, None] + V * ref.U32) + \
        (g.double() * rest * 2 * rel)[:, None] * W[y].abs()
    edh = edh + ref.HALF[torch.bfloat16] * (dh.abs() + edh) + ref.TINY

    t = y.int()
    for name, got in (("alone", ops.head_cross_entropy(h, *w, t, group_size=group, bits=bits)),
                      ("with dh", ops.head_cross_entropy(h, *w, t, grad=True, grad_loss=g,
                                                         group_size=group, bits=bits))):
        assert (got[0] >= 0).all()
        ref.check(got[0], loss, eloss, f"loss {name}")
        ref.check(got[1], lse, logit_error(h, W, 1.0) + eloss + 4 * ref.U32 * lse.abs(), f"lse {name}")
    ref.check(got[2], dh, edh, "dh")
    ops.device_error()


@pytest.mark.parametrize("T", [1.0, 2.0])
@pytest.mark.parametrize("M,V,K", [(40, 1500, 256), (150, 30000, 256), (1100, 24000, 256)])
def test_distill_of_rows_that_agree_with_the_teacher(gpu, M, V, K, T):
    """The teacher's logits are the row's own but for noise of 0, 1e-3 or 0.1, and its entries take
    nearly everything: the divergence is a sum of squares, plus what is left to the others.  With
    D_v the error of a logit it moves by sum_v (p_v - q_v) D_v and by squares of D."""
    announce(f"agreeing rows {M}x{V}x{K}, T {T}")
    gen = torch.Generator().manual_seed(M)
    w = ref.quant(gen, (V,), K, 4, 64, gpu)
    W = ref.values(*w, 4, 64)
    a = torch.randint(0, V - 200, (M,), generator=gen)
    # The other entry in the same tile for every second row.
    b = a + torch.where(torch.arange(M) % 2 == 0, torch.ones_like(a),
                        torch.randint(150, 200, (M,), generator=gen))
    c = (a + 17) % V
    ids = torch.stack([a, b, c], 1).to(gpu)
    E = W[ids[:, :2]]                                  # [M, 2, K]
    both = torch.linalg.solve(E @ E.transpose(1, 2).contiguous(),
                              torch.ones(M, 2, 1, dtype=torch.float64, device=gpu))
    lead = torch.linspace(0, 60 * T, M, dtype=torch.float64, device=gpu)
    h = ((both * E).sum(1) * lead[:, None]).bfloat16()

    logits = h.double() @ W.T / T
    logp = torch.log_softmax(logits, -1).gather(1, ids)
    noise = torch.tensor([0, 1e-3, 0.1], dtype=torch.float64)[torch.arange(M) % 3]
    noise = noise[:, None] * torch.randn(M, 3, generator=gen, dtype=torch.float64)
    teacher = (T * (logits.gather(1, ids) + noise.to(gpu))).float()
    logq = torch.log_softmax(teacher.double() / T, -1)
    p, q, d = logp.exp(), logq.exp(), logq - logp
    rest = logits.scatter(1, ids, -torch.inf)
    rest = (torch.logsumexp(rest, -1) - torch.logsumexp(logits, -1)).exp()
    loss = T * T * ((q * (d + torch.expm1(-d))).sum(-1) + rest)
    assert loss.min() < 1e-8 and loss.max() > 0.1
    delta = 2 * logit_error(h, W, T) + 8 * ref.U32 * teacher.double().abs().amax(-1) / T
    apart = (p - q).abs().sum(-1) + rest
    eloss = T * T * (apart * (2 * delta + sums_error(V)) + 4 * delta ** 2) + 256 * ref.U32 * loss
    # 64 bits of log p and log q differ by their own roundings.
    eloss = eloss + T * T * 1e-14 * logits.abs().amax(-1)
    assert (eloss < 0.5 * loss).double().mean() > 0.5  # the bound says something

    ecoef = 2 * delta[:, None] * (p * (1 - p) + q * (1 - q)) + 64 * ref.U32 * (p - q).abs() + \
        64 * ref.U32 * (p * (1 - p) + q * (1 - q))
    full = torch.softmax(logits, -1).scatter(1, ids, 0.0)
    dh = T * (full @ W + ((p - q)[..., None] * W[ids]).sum(1))
    edh = T * ((full @ W.abs()) * (ref.HALF[torch.bfloat16] + 2 * delta + sums_error(V))[:, None] +
               (ecoef[..., None] * W[ids].abs()).sum(1) + 8 * ref.U32 *
               ((p - q).abs()[..., None] * W[ids].abs()).sum(1))
    edh = edh + ref.HALF[torch.bfloat16] * (dh.abs() + edh) + ref.TINY

    i = ids.int()
    got = ops.head_distill(h, *w, i, teacher, temperature=T, grad=True)
    only = ops.head_distill(h, *w, i, teacher, temperature=T)
    for name, loss_got in (("with dh", got[0]), ("alone", only[0])):
        assert (loss_got >= 0).all()
        ref.check(loss_got, loss, eloss, f"loss {name}")
    ref.check(got[2], dh, edh, "dh")
    ops.device_error()


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("M", [3, 130, 1900])
def test_every_token_is_wanted(gpu, M, grad):
    """No token is left to a tile, or to the row."""
    announce(f"every token wanted, {M} rows")
    gen = torch.Generator().manual_seed(M)
    for V in (1, 3, 64):
        w = ref.quant(gen, (V,), 64, 4, 64, gpu)
        h = torch.randn(M, 64, generator=gen).bfloat16().to(gpu)
        ids = torch.arange(V, dtype=torch.int32, device=gpu).repeat(M, 1)
        t = torch.randn(M, V, generator=gen).to(gpu)
        logits = h.double() @ ref.values(*w, 4, 64).T
        logp, logq = logits.log_softmax(-1), t.double().log_softmax(-1)
        loss = (logq.exp() * (logq - logp)).sum(-1)
        got = ops.head_distill(h, *w, ids, t, grad=grad)
        d = 2 * logit_error(h, ref.values(*w, 4, 64), 1.0) + 64 * ref.U32 * (1 + t.double().abs().amax(-1))
        ref.check(got[0], loss, 2 * d + 1e-14, "loss")
        ref.check(got[1], torch.logsumexp(logits, -1), d, "lse")
        if grad:
            W = ref.values(*w, 4, 64)
            e = (2 * d)[:, None] * W.abs().sum(0)
            dh = (logp.exp() - logq.exp()) @ W
            ref.check(got[2], dh, e + ref.HALF[torch.bfloat16] * (dh.abs() + e), "dh")
