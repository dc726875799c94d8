"""64-bit references and error bounds of the adapters beside quantized products (test side, torch).

u = 2^-24: an fp32 sum of n products is off by at most (n + 2) u of their magnitudes' sum, whatever
its order.  A value that enters a matrix product as two bf16 values keeps 2^-17 of itself: the
first is off by 2^-9 at most, and the second, which holds that, by 2^-9 of it (2^-18; twice that where
the first rounding crossed a power of two).
"""
import torch

import grad_ref as R

SPLIT = 2.0 ** -17
# The third of three values holds what the first two leave to 2^-9 of it: all bits, but for a
# last unit.
SPLIT3 = 2.0 ** -24


def make(gen, M, N, K, E, r, bits, group, dev, adapters="runs"):
    w = R.quant(gen, (N,), K, bits, group, dev)
    x = torch.randn(M, K, generator=gen).bfloat16().to(dev)
    a = (torch.randn(E, r, K, generator=gen) / K ** 0.5).bfloat16().to(dev)
    b = (torch.randn(E, N, r, generator=gen) * 0.5 / r ** 0.5).bfloat16().to(dev)
    s = (0.5 + torch.rand(E, generator=gen)).to(dev)
    if adapters == "runs":
        ids = (torch.arange(M) * (E + 1) // max(M, 1)) - 1 if E > 1 else torch.zeros(M)
    elif adapters == "mixed":
        ids = torch.randint(-1, E, (M,), generator=gen)
    elif adapters == "none":
        ids = torch.full((M,), -1)
    else:
        ids = torch.full((M,), adapters)
    return x, w, a, b, ids.int().to(dev), s


def product(x, W):
    """x @ W^T in 64 bits and the bound of its fp32 sum."""
    x = x.double()
    return x @ W.T, (W.shape[1] + 64) * R.U32 * (x.abs() @ W.abs().T)


def _shrink(p, v):
    """P @ V^T and its bound."""
    t = p @ v.T
    return t, (p.shape[1] + 8) * R.U32 * (p.abs() @ v.abs().T)


def delta(p, ids, v1, v2, s):
    """s_e (P V1_e^T) V2_e^T of each row and its bound; zero for rows without adapter."""
    out = torch.zeros(p.shape[0], v2.shape[1], dtype=torch.float64, device=p.device)
    err = torch.zeros_like(out)
    for e in range(v1.shape[0]):
        on = (ids == e).nonzero()[:, 0]
        if not len(on):
            continue
        t, et = _shrink(p[on].double(), v1[e].double())
        se, V = float(s[e]), v2[e].double()
        out[on] = se * (t @ V.T)
        err[on] = abs(se) * ((et + (SPLIT + 2 * R.U32) * t.abs()) @ V.abs().T +
                             (2 * V.shape[1] + 8) * R.U32 * (t.abs() @ V.abs().T))
    return out, err


def outer(p, q, ids, v, s, E):
    """s_e sum over e's rows of (Q V_e^T)^T P: [E, r, C] and its bound."""
    r, C = v.shape[1], p.shape[1]
    g = torch.zeros(E, r, C, dtype=torch.float64, device=p.device)
    err = torch.zeros_like(g)
    for e in range(E):
        on = (ids == e).nonzero()[:, 0]
        if not len(on):
            continue
        t, et = _shrink(q[on].double(), v[e].double())
        P, se = p[on].double(), float(s[e])
        g[e] = se * (t.T @ P)
        err[e] = abs(se) * ((et + (SPLIT3 + 2 * R.U32) * t.abs()).T @ P.abs() +
                            (3 * len(on) + 64) * R.U32 * (t.abs().T @ P.abs()))
    return g, err + R.TINY


def rounded(y, err):
    """The bound of a bf16 value of y with an error of err."""
    return err + R.HALF[torch.bfloat16] * (y.abs() + err) + R.TINY
