"""64-bit references and error bounds for the training operators (test side, torch).

The bounds count roundings.  With u = 2^-24 an fp32 sum of n products is off by at most
(n + 2) u times the sum of their magnitudes, whatever its order; a rounding to type t is off by
at most eps(t) / 2 of the value (bf16: 2^-8).
"""
from __future__ import annotations

import torch

U32 = 2.0 ** -24
HALF = {torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2, torch.float32: U32}
TINY = 1e-37  # below fp32's normal range


def quant(gen, lead, K, bits, group, device="cpu"):
    """A random quantized weight triple in the distributions of the benchmark."""
    w = torch.randint(-2**31, 2**31, (*lead, K * bits // 32), generator=gen, dtype=torch.int64)
    lo, hi, mid = (0.002, 0.02, 8) if bits == 4 else (1e-4, 2e-3, 128)
    s = (torch.rand(*lead, K // group, generator=gen) * (hi - lo) + lo).bfloat16()
    b = -mid * s.float()
    if bits == 4:
        b = b + 1e-3 * torch.randn(b.shape, generator=gen)
    return w.int().to(device), s.to(device), b.bfloat16().to(device)


def values(w, s, b, bits, group):
    """deq(W) as dequantize defines it, in float64."""
    at = torch.arange(0, 32, bits, device=w.device, dtype=torch.int32)
    q = ((w.unsqueeze(-1) >> at) & ((1 << bits) - 1)).reshape(*s.shape, group).float()
    v = (q * s.float().unsqueeze(-1)).bfloat16().float() + b.float().unsqueeze(-1)
    return v.bfloat16().double().reshape(*w.shape[:-1], -1)


def head(h, W, ids, q, keep, temperature, g):
    """loss, lse and dh of rows with wanted distribution q [M, k] over ids (absent entries: q
    0, id 0) and their bounds.  keep [M] is False for rows without a wanted entry."""
    h, T = h.double(), float(temperature)
    M, K = h.shape
    logits = h @ W.T / T
    lse = torch.logsumexp(logits, -1)
    logp = logits - lse[:, None]
    sel = logp.gather(1, ids)
    ent = torch.where(q > 0, q * q.clamp(min=1e-300).log(), torch.zeros_like(q))
    loss = torch.where(keep, T * T * (ent - torch.where(q > 0, q * sel, torch.zeros_like(q))).sum(-1),
                       torch.zeros_like(lse))
    p = logp.exp()
    wanted = torch.zeros_like(p).scatter_add_(1, ids, q)
    scale = torch.where(keep, g.double() * T, torch.zeros_like(lse))
    dh = scale[:, None] * ((p - wanted) @ W)
    # A logit: an fp32 sum of K products, the scaling, and the constants log2 e and ln 2 in
    # fp32 (4 more roundings of its size).  lse: the logits' error, a sum of at most V + 512
    # terms in fp32 (each tile's and over tiles), exp2 and log2 to 2 units each.
    V = W.shape[0]
    size = (h.abs() @ W.abs().T).amax(-1) / T
    el = (K + 8) * U32 * size
    es = (min(V, 2048) + 64) * U32
    elog = el + es + 8 * U32 * (lse.abs() + size)
    # The wanted distribution's own fp32 arithmetic: a few units of log q and log p.
    mag = (q * (q.clamp(min=1e-300).log().abs() + sel.abs())).sum(-1)
    eloss = T * T * (2 * elog + 100 * U32 * (1 + mag))
    # dh: e to bf16 once (2^-8 of each term but the wanted ones'), p through the logits' error,
    # the fp32 sums, and the result's rounding.
    pabs = p @ W.abs()
    wabs = wanted @ W.abs()
    rest = p.scatter(1, ids, torch.zeros_like(q)) @ W.abs()
    ed = scale.abs()[:, None] * (HALF[torch.bfloat16] * rest + (2 * elog + 1e-5)[:, None] *
                                 (pabs + wabs) + (V + 64) * U32 * (pabs + wabs))
    ed = ed + HALF[torch.bfloat16] * (dh.abs() + ed) + TINY
    return (loss, eloss), (lse, elog), (dh, ed)


def teacher_q(ids, teacher, V, temperature):
    """The wanted distribution of a teacher's entries (ids clamped, absent ones 0) and which
    rows have any."""
    on = (ids >= 0) & (ids < V)
    t = torch.where(on, teacher.double() / temperature, torch.full_like(teacher, -torch.inf,
                                                                         dtype=torch.float64))
    top = t.amax(-1, keepdim=True)
    keep = top[:, 0] > -torch.inf
    e = torch.where(keep[:, None], (t - top).exp(), torch.zeros_like(t))
    q = torch.where(keep[:, None], e / e.sum(-1, keepdim=True).clamp(min=1e-300), e)
    return torch.where(on, ids, torch.zeros_like(ids)).long(), q, keep


def product(dy, W):
    """dy @ W in 64 bits and its bound as bf16."""
    y = dy.double() @ W
    e = (W.shape[0] + 2) * U32 * (dy.double().abs() @ W.abs())
    return y, e + HALF[torch.bfloat16] * (y.abs() + e) + TINY


def check(got, ref, bound, what=""):
    got = got.double()
    assert got.shape == ref.shape, f"{what}: {tuple(got.shape)} against {tuple(ref.shape)}"
    bad = ~((got - ref).abs() <= bound)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: "
                             f"{float(got[i])} against {float(ref[i])} +- {float(bound[i])}")
