"""Adapters beside quantized products, and their gradients, against 64-bit references."""
import pytest
import torch

import grad_ref as R
import lora_ref as L
from fastmlx_amd import FmxqError, ops
from gpu_util import announce

pytestmark = pytest.mark.gpu


def check_forward(x, w, a, b, ids, s, group, bits):
    y = ops.quantized_matmul_lora(x, *w, a, b, ids, s, group, bits)
    K, N = x.shape[-1], w[0].shape[0]
    flat = x.reshape(-1, K)
    base, eb = L.product(flat, R.values(*w, bits, group))
    d, e = L.delta(flat, ids.flatten(), a, b, s)
    R.check(y.reshape(-1, N), base + d, L.rounded(base + d, eb + e), "y")
    return y


FORWARD = [
    # M, N, K, E, r, bits, group, adapters
    (1, 256, 256, 1, 8, 4, 64, "runs"), (1, 37, 512, 3, 16, 8, 64, 1), (1, 264, 128, 2, 128, 4, 128, 0),
    (5, 130, 96, 4, 24, 4, 32, "mixed"), (33, 72, 256, 5, 40, 8, 32, "mixed"), (64, 1000, 512, 8, 16, 4, 64, "mixed"),
    (128, 512, 256, 7, 64, 4, 64, "mixed"), (129, 520, 256, 7, 16, 4, 64, "mixed"), (130, 131, 128, 1, 8, 4, 64, "runs"),
    (200, 640, 320, 1, 32, 4, 64, "runs"), (300, 1032, 512, 6, 64, 4, 64, "runs"), (301, 136, 128, 40, 24, 8, 64, "mixed"),
    (513, 520, 256, 3, 128, 4, 64, "runs"), (700, 96, 2048, 2, 56, 4, 64, "mixed"), (1100, 260, 256, 12, 16, 4, 64, "mixed"),
    (150, 72, 64, 4, 16, 4, 64, "none"), (20, 72, 64, 4, 16, 4, 64, "none"),
]


@pytest.mark.parametrize("M,N,K,E,r,bits,group,ids", FORWARD)
def test_forward(gpu, M, N, K, E, r, bits, group, ids):
    announce(f"lora forward {M} {N} {K} {E} {r} {bits} {group} {ids}")
    gen = torch.Generator().manual_seed(M + N + r)
    check_forward(*L.make(gen, M, N, K, E, r, bits, group, gpu, ids), group, bits)


def check_grad(x, w, a, b, ids, s, group, bits, dy):
    dx, da, db = ops.quantized_matmul_lora_grad(dy, x, *w, a, b, ids, s, group, bits)
    K, N, E = x.shape[-1], w[0].shape[0], a.shape[0]
    X, D, I = x.reshape(-1, K), dy.reshape(-1, N), ids.flatten()
    W = R.values(*w, bits, group)
    base, eb = L.product(D, W.T)
    at, bt = a.transpose(1, 2).contiguous(), b.transpose(1, 2).contiguous()
    d, e = L.delta(D, I, bt, at, s)
    want = base + d
    R.check(dx.reshape(-1, K), want, L.rounded(want, eb + e), "dx")
    ga, ea = L.outer(X, D, I, bt, s, E)
    R.check(da, ga, ea, "da")
    gb, eb = L.outer(D, X, I, a, s, E)
    R.check(db, gb.transpose(1, 2), eb.transpose(1, 2), "db")
    return dx, da, db


GRAD = [
    (1, 256, 256, 1, 8, 4, 64, "runs"), (2, 37, 512, 3, 16, 8, 64, "mixed"), (31, 264, 128, 2, 128, 4, 128, "mixed"),
    (33, 130, 96, 4, 24, 4, 32, "mixed"), (64, 1000, 512, 8, 16, 4, 64, "mixed"), (129, 520, 256, 7, 64, 4, 64, "mixed"),
    (200, 131, 128, 1, 8, 4, 64, "runs"), (300, 1032, 512, 6, 32, 4, 64, "runs"), (301, 136, 128, 40, 24, 8, 64, "mixed"),
    (513, 520, 256, 1, 128, 4, 64, "runs"), (1100, 260, 256, 3, 16, 4, 64, "mixed"), (1500, 96, 1024, 1, 40, 4, 64, "runs"),
    (150, 72, 64, 4, 16, 4, 64, "none"), (700, 72, 64, 1, 16, 4, 64, "none"), (900, 4104, 64, 2, 16, 4, 64, "runs"),
]


@pytest.mark.parametrize("M,N,K,E,r,bits,group,ids", GRAD)
def test_grad(gpu, M, N, K, E, r, bits, group, ids):
    announce(f"lora grad {M} {N} {K} {E} {r} {bits} {group} {ids}")
    gen = torch.Generator().manual_seed(M + N + r)
    c = L.make(gen, M, N, K, E, r, bits, group, gpu, ids)
    dy = torch.randn(M, N, generator=gen).bfloat16().to(gpu)
    check_grad(*c, group, bits, dy)


def test_one_adapter_with_rows_of_none(gpu):
    """One adapter takes no sort: rows without it, infinities among them, stay out of its gradients."""
    gen = torch.Generator().manual_seed(3)
    x, w, a, b, ids, s = L.make(gen, 300, 264, 256, 1, 16, 4, 64, gpu, "mixed")
    dy = torch.randn(300, 264, generator=gen).bfloat16().to(gpu)
    check_grad(x, w, a, b, ids, s, 64, 4, dy)
    clean = ops.quantized_matmul_lora_grad(dy, x, *w, a, b, ids, s)
    off = (ids < 0).nonzero()[:, 0]
    x[off[0]] = float("inf")
    dy[off[1]] = float("nan")
    _, da, db = ops.quantized_matmul_lora_grad(dy, x, *w, a, b, ids, s)
    assert torch.equal(da, clean[1]) and torch.equal(db, clean[2])


@pytest.mark.parametrize("M", [40, 300])
def test_bad_rows_and_adapters_stay_alone(gpu, M):
    gen = torch.Generator().manual_seed(4)
    x, w, a, b, ids, s = L.make(gen, M, 264, 256, 3, 16, 4, 64, gpu, "mixed")
    y = ops.quantized_matmul_lora(x, *w, a, b, ids, s)
    dy = torch.randn(M, 264, generator=gen).bfloat16().to(gpu)
    g = ops.quantized_matmul_lora_grad(dy, x, *w, a, b, ids, s)
    a2, b2 = a.clone(), b.clone()
    a2[1, 3, 5], b2[1, 7, 2] = float("inf"), float("nan")
    others = ids != 1
    assert torch.equal(ops.quantized_matmul_lora(x, *w, a2, b2, ids, s)[others], y[others])
    dx, da, db = ops.quantized_matmul_lora_grad(dy, x, *w, a2, b2, ids, s)
    assert torch.equal(dx[others], g[0][others])
    for e in (0, 2):
        assert torch.equal(da[e], g[1][e]) and torch.equal(db[e], g[2][e])
    row = int((ids == 1).nonzero()[0])
    x2 = x.clone()
    x2[row] = float("nan")
    keep = torch.arange(M, device=gpu) != row
    assert torch.equal(ops.quantized_matmul_lora(x2, *w, a, b, ids, s)[keep], y[keep])
    assert ops.quantized_matmul_lora(x2, *w, a, b, ids, s)[row].isnan().all()


@pytest.mark.parametrize("M,E", [(9, 2), (300, 2), (300, 1)])
def test_an_adapter_past_the_last_is_none_and_reported(gpu, M, E):
    gen = torch.Generator().manual_seed(5)
    x, w, a, b, ids, s = L.make(gen, M, 136, 128, E, 8, 4, 64, gpu, "mixed")
    ids[M // 2] = E
    ids[3] = -2**31
    ops.device_error()
    check_forward(x, w, a, b, ids, s, 64, 4)
    with pytest.raises(FmxqError):
        ops.device_error()
    dy = torch.randn(M, 136, generator=gen).bfloat16().to(gpu)
    check_grad(x, w, a, b, ids, s, 64, 4, dy)
    with pytest.raises(FmxqError):
        ops.device_error()
    ops.quantized_matmul_lora(x, *w, a, b, ids.clamp(max=E - 1), s)
    ops.device_error()


def test_batches_and_alignment(gpu):
    gen = torch.Generator().manual_seed(6)
    for M, N in ((6, 136), (200, 136), (200, 131)):
        x, w, a, b, ids, s = L.make(gen, M, N, 128, 3, 8, 4, 64, gpu, "mixed")
        dy = torch.randn(M, N, generator=gen).bfloat16().to(gpu)
        y = check_forward(x, w, a, b, ids, s, 64, 4)
        shaped = (2, M // 2)
        assert torch.equal(ops.quantized_matmul_lora(x.view(*shaped, 128), *w, a, b, ids.view(shaped), s),
                           y.view(*shaped, N))
        g = check_grad(x, w, a, b, ids, s, 64, 4, dy)
        buf = torch.empty(M * N + 1, dtype=torch.bfloat16, device=gpu)
        moved = buf[1:].view(M, N).copy_(dy)
        h = ops.quantized_matmul_lora_grad(moved.view(*shaped, N), x.view(*shaped, 128), *w, a, b,
                                           ids.view(shaped), s)
        for p, q in zip(g, h):
            assert torch.equal(p.flatten(), q.flatten())


def test_no_rows_and_no_columns(gpu):
    gen = torch.Generator().manual_seed(7)
    x, w, a, b, ids, s = L.make(gen, 4, 64, 64, 2, 8, 4, 64, gpu, "mixed")
    assert ops.quantized_matmul_lora(x[:0], *w, a, b, ids[:0], s).shape == (0, 64)
    dx, da, db = ops.quantized_matmul_lora_grad(torch.empty(0, 64, dtype=torch.bfloat16, device=gpu), x[:0], *w,
                                                a, b, ids[:0], s)
    assert dx.shape == (0, 64) and not da.any() and not db.any()
    none = tuple(t[:0] for t in w)
    dx, da, db = ops.quantized_matmul_lora_grad(torch.empty(4, 0, dtype=torch.bfloat16, device=gpu), x, *none, a,
                                                b[:, :0].contiguous(), ids, s)
    assert not dx.any() and not da.any() and db.shape == (2, 0, 8)


def test_gradients_against_differences(gpu):
    """In 64 bits over the plain formula: the operator's gradients are that formula's."""
    gen = torch.Generator().manual_seed(8)
    x, w, a, b, ids, s = L.make(gen, 6, 24, 64, 2, 8, 4, 64, "cpu", "mixed")
    W = R.values(*w, 4, 64)
    dy = torch.randn(6, 24, generator=gen).bfloat16()

    def loss(x, a, b):
        y = x @ W.T
        for m in range(6):
            if ids[m] >= 0:
                e = int(ids[m])
                y[m] += float(s[e]) * (b[e] @ (a[e] @ x[m]))
        return (y * dy.double()).sum()

    args = [t.double() for t in (x, a, b)]
    got = ops.quantized_matmul_lora_grad(*(t.to(gpu) for t in (dy, x, *w, a, b, ids, s)))
    for i, g in enumerate(got):
        g = g.double().cpu()
        d = torch.randn(g.shape, generator=gen, dtype=torch.float64)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + 1e-4 * d, args[i] - 1e-4 * d
        slope = (loss(*up) - loss(*down)) / 2e-4  # linear in each: exact but for rounding
        size = (g.abs() * d.abs()).sum()
        assert abs(float((g * d).sum() - slope)) <= (2.0 ** -8 if i == 0 else 2.0 ** -15) * float(size)


def step(c, dy):
    x, w, a, b, ids, s = c
    y = ops.quantized_matmul_lora(x, *w, a, b, ids, s)
    dx, da, db = ops.quantized_matmul_lora_grad(dy, x, *w, a, b, ids, s)
    clipped, norm = ops.clip_grad_norm([da, db], 0.5)
    return [y, dx, *clipped, norm]


@pytest.mark.parametrize("M", [20, 300])
def test_streams_and_graphs(gpu, M):
    """The same bits on another stream and from a graph replayed among eager work."""
    gen = torch.Generator().manual_seed(9)
    c = L.make(gen, M, 520, 256, 3, 16, 4, 64, gpu, "mixed")
    dy = torch.randn(M, 520, generator=gen).bfloat16().to(gpu)
    want = step(c, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for p, q in zip(step(c, dy), want):
            assert torch.equal(p, q)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(c, dy)
    for k in range(3):
        x = torch.randn(c[0].shape, generator=gen).bfloat16().to(gpu)
        c[0].copy_(x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, step(c, dy)):
            assert torch.equal(p, q), k


def test_refuses(gpu):
    gen = torch.Generator().manual_seed(10)
    x, w, a, b, ids, s = L.make(gen, 4, 64, 64, 2, 8, 4, 64, gpu, "mixed")
    f = ops.quantized_matmul_lora
    with pytest.raises(ValueError):
        f(x, *w, a, b, ids[:3], s)
    with pytest.raises(ValueError):
        f(x, *w, a[:1], b, ids, s)
    with pytest.raises(ValueError):
        f(x, *w, a, b[:, :, :4], ids, s)
    with pytest.raises(TypeError):
        f(x, *w, a, b, ids.long(), s)
    with pytest.raises(TypeError):
        f(x, *w, a.float(), b, ids, s)
    with pytest.raises(TypeError):
        f(x, *w, a, b, ids, s.double())
    with pytest.raises(ValueError):
        f(x, *w, a, b, ids, s.cpu())
    with pytest.raises(FmxqError):
        f(x, *w, a[:, :4].contiguous(), b[:, :, :4].contiguous(), ids, s)
    dy = torch.zeros(4, 64, dtype=torch.bfloat16, device=gpu)
    with pytest.raises(ValueError):
        ops.quantized_matmul_lora_grad(dy[:, :32].contiguous(), x, *w, a, b, ids, s)
    with pytest.raises(ValueError):
        ops.quantized_matmul_lora_grad(dy.t(), x, *w, a, b, ids, s)
