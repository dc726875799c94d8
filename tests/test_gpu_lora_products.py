"""Adapters beside each of the products that they enter: few rows, tiles and their edges, pieces of a cut
tile, a panel; more adapters and rows than one block sorts; a step of them all."""
import pytest
import torch

import grad_ref as R
import lora_ref as L
from fastmlx_amd import ops
from gpu_util import announce
from test_gpu_clip import check as check_clip
from test_gpu_logprobs import Ref, check_grad as check_logprobs_grad
from test_gpu_lora import check_forward, check_grad

pytestmark = pytest.mark.gpu

PRODUCTS = [
    # M, N, K, E, r, bits, group, adapters
    # Many rows of widths that are multiples of 256: whole tiles and cut ones, tiles' last rows and columns.
    (2048, 4096, 1024, 3, 16, 4, 64, "mixed"), (2049, 4104, 512, 1, 72, 4, 64, "runs"),
    (1030, 4104, 1024, 9, 128, 8, 32, "mixed"), (1300, 4104, 768, 2, 8, 4, 128, "runs"),
    (200, 8200, 2048, 4, 64, 4, 32, "mixed"), (4096, 2056, 512, 5, 40, 8, 128, "runs"),
    (1300, 4104, 768, 3, 104, 8, 64, "mixed"), (1100, 4104, 1024, 2, 16, 4, 64, "none"),
    # Other widths: tiles straight from the weights, with and without a panel of them.
    (1000, 4100, 320, 4, 72, 4, 64, "mixed"), (500, 8260, 320, 2, 16, 8, 32, "runs"),
    (300, 20001, 320, 3, 8, 4, 32, "mixed"), (1900, 4102, 320, 3, 128, 4, 64, "mixed"),
    (2000, 4101, 96, 1, 24, 8, 32, "runs"), (1900, 4102, 320, 2, 16, 4, 64, "none"),
    # ... in parts of the contraction, and more weights than one panel holds.
    (1000, 4100, 1088, 3, 16, 4, 64, "mixed"), (1800, 2052, 1088, 2, 40, 8, 32, "mixed"),
    (1793, 66004, 4128, 2, 8, 4, 32, "runs"),
    # Few rows of long ones.
    (3, 40, 99968, 2, 8, 4, 64, "mixed"), (70, 72, 99968, 2, 8, 8, 64, "mixed"),
]


@pytest.mark.parametrize("M,N,K,E,r,bits,group,ids", PRODUCTS)
def test_products(gpu, M, N, K, E, r, bits, group, ids):
    announce(f"lora product {M} {N} {K} {E} {r} {bits} {group} {ids}")
    gen = torch.Generator().manual_seed(M + N + r)
    check_forward(*L.make(gen, M, N, K, E, r, bits, group, gpu, ids), group, bits)


@pytest.mark.parametrize("M", range(1, 19))
def test_few_rows(gpu, M):
    """Every number of rows around the product for few; outputs that end inside a block, a row that ends
    inside its step."""
    announce(f"lora few rows {M}")
    gen = torch.Generator().manual_seed(M)
    for N, K, bits, group in ((17, 64, 4, 64), (301, 320, 4, 32), (129, 1088, 8, 32), (40, 2048, 8, 128)):
        check_forward(*L.make(gen, M, N, K, 3, 16, bits, group, gpu, "mixed"), group, bits)


def test_few_rows_of_much_weight(gpu):
    """Above 8 rows large weights go another way."""
    announce("lora 9 and 16 rows, 8200 x 4352")
    gen = torch.Generator().manual_seed(1)
    for M in (8, 9, 16):
        check_forward(*L.make(gen, M, 8200, 4352, 2, 8, 4, 64, gpu, "mixed"), 64, 4)


@pytest.mark.parametrize("M,E", [(700, 511), (700, 512), (700, 2048), (16384, 3), (16385, 3)])
def test_many_adapters_and_rows(gpu, M, E):
    announce(f"lora sort {M} {E}")
    gen = torch.Generator().manual_seed(M + E)
    c = L.make(gen, M, 72, 64, E, 8, 4, 64, gpu, "mixed")
    check_forward(*c, 64, 4)
    dy = torch.randn(M, 72, generator=gen).bfloat16().to(gpu)
    check_grad(*c, 64, 4, dy)


@pytest.mark.parametrize("M,N,K", [(2048, 4104, 512), (1900, 4102, 320), (1000, 4100, 320), (16, 520, 320)])
def test_bad_rows_and_adapters_stay_alone(gpu, M, N, K):
    announce(f"lora bad {M} {N} {K}")
    gen = torch.Generator().manual_seed(4)
    x, w, a, b, ids, s = L.make(gen, M, N, K, 3, 72, 4, 64, gpu, "mixed")
    y = ops.quantized_matmul_lora(x, *w, a, b, ids, s)
    a2, b2 = a.clone(), b.clone()
    a2[1, 3, 5], a2[1, 70, 5], b2[1, 7, 2], b2[1, 8, 71] = (float("inf"),) * 2 + (float("nan"),) * 2
    others = ids != 1
    assert torch.equal(ops.quantized_matmul_lora(x, *w, a2, b2, ids, s)[others], y[others])
    row = int((ids == 1).nonzero()[0])
    x2 = x.clone()
    x2[row] = float("nan")
    keep = torch.arange(M, device=gpu) != row
    got = ops.quantized_matmul_lora(x2, *w, a, b, ids, s)
    assert torch.equal(got[keep], y[keep]) and got[row].isnan().all()


@pytest.mark.parametrize("M,N,K", [(200, 8200, 2048), (1900, 4102, 320), (12, 520, 320)])
def test_streams_and_graphs(gpu, M, N, K):
    """Products whose last block waits for others: the same bits at every replay."""
    announce(f"lora graph {M} {N} {K}")
    gen = torch.Generator().manual_seed(9)
    c = L.make(gen, M, N, K, 3, 16, 4, 64, gpu, "mixed")
    want = ops.quantized_matmul_lora(*c[:1], *c[1], *c[2:])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.quantized_matmul_lora(*c[:1], *c[1], *c[2:]), want)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = ops.quantized_matmul_lora(*c[:1], *c[1], *c[2:])
    for k in range(3):
        c[0].copy_(torch.randn(M, K, generator=gen).bfloat16())
        c[4].copy_(torch.randint(-1, 3, (M,), generator=gen))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.quantized_matmul_lora(*c[:1], *c[1], *c[2:])), k


@pytest.mark.parametrize("M,N,K", [(3, 72, 256), (40, 72, 256), (300, 72, 256), (2048, 4104, 512), (1000, 4100, 320),
                                   (1900, 4102, 320)])
def test_any_alignment_of_scales(gpu, M, N, K):
    """Scales, biases and the adapters' numbers and scales at any multiple of their size: the same bits."""
    announce(f"lora scales' alignment {M} {N} {K}")
    gen = torch.Generator().manual_seed(5)
    x, w, a, b, ids, s = L.make(gen, M, N, K, 3, 16, 4, 64, gpu, "mixed")

    def moved(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=gpu)
        return buf[1:].view(t.shape).copy_(t)

    w2 = (w[0], moved(w[1]), moved(w[2]))
    assert torch.equal(ops.quantized_matmul_lora(x, *w2, a, b, moved(ids), moved(s)),
                       ops.quantized_matmul_lora(x, *w, a, b, ids, s))
    dy = torch.randn(M, N, generator=gen).bfloat16().to(gpu)
    for p, q in zip(ops.quantized_matmul_lora_grad(dy, x, *w2, a, b, moved(ids), moved(s)),
                    ops.quantized_matmul_lora_grad(dy, x, *w, a, b, ids, s)):
        assert torch.equal(p, q)
    t = torch.randint(0, N, (M, 1), generator=gen).int().to(gpu)
    for p, q in zip(ops.head_logprobs(x, *w2, moved(t), top=5), ops.head_logprobs(x, *w, t, top=5)):
        assert torch.equal(p, q)


def test_a_dirty_workspace(gpu):
    """What a workspace held before makes no difference: through the C entry points, with the workspace
    filled with NaN bits and with ones, and 16 bytes of guard behind it."""
    import ctypes

    from fastmlx_amd._lib import load

    lib = load()
    gen = torch.Generator().manual_seed(6)
    for M, N, K, E in ((5, 72, 256, 2), (40, 72, 256, 2), (300, 72, 256, 3), (700, 72, 64, 600), (200, 8200, 2048, 3),
                       (1000, 4100, 1088, 1)):
        announce(f"dirty workspace {M} {N} {K} {E}")
        x, w, a, b, ids, s = L.make(gen, M, N, K, E, 8, 4, 64, gpu, "mixed")
        dy = torch.randn(M, N, generator=gen).bfloat16().to(gpu)
        want = [ops.quantized_matmul_lora(x, *w, a, b, ids, s), *ops.quantized_matmul_lora_grad(dy, x, *w, a, b, ids, s)]
        size = ctypes.c_size_t()
        common = [t.data_ptr() for t in (x, *w, a, b, ids, s)]
        st = torch.cuda.current_stream().cuda_stream
        for fill in (0xFF, 0x01):
            got = [torch.empty_like(t) for t in want]
            assert lib.fmxq_quantized_matmul_lora_workspace(M, N, K, E, 8, ctypes.byref(size)) == 0
            ws = torch.full((size.value + 16,), fill, dtype=torch.uint8, device=gpu)
            assert lib.fmxq_quantized_matmul_lora(*common, got[0].data_ptr(), M, N, K, E, 8, 64, 4, ws.data_ptr(),
                                                  size.value, st) == 0
            assert bool((ws[size.value:] == fill).all())
            assert lib.fmxq_quantized_matmul_lora_grad_workspace(M, N, K, E, 8, ctypes.byref(size)) == 0
            ws = torch.full((size.value + 16,), fill, dtype=torch.uint8, device=gpu)
            assert lib.fmxq_quantized_matmul_lora_grad(dy.data_ptr(), *common, *(t.data_ptr() for t in got[1:]), M, N, K,
                                                       E, 8, 64, 4, ws.data_ptr(), size.value, st) == 0
            assert bool((ws[size.value:] == fill).all())
            for p, q in zip(got, want):
                assert torch.equal(p, q)


def policy_step(x, w, a, b, ids, s, head, tokens, adv, beta, max_norm):
    """A layer with adapters, its rows' log probabilities of tokens and entropy, and the clipped gradients
    of  -sum adv logp - beta sum entropy."""
    h = ops.quantized_matmul_lora(x, *w, a, b, ids, s)
    scores = ops.head_logprobs(h, *head, tokens)
    c = torch.full_like(scores[1], -beta)
    dh = ops.head_logprobs_grad(h, *head, tokens, *scores, -adv, grad_entropy=c)
    dx, da, db = ops.quantized_matmul_lora_grad(dh, x, *w, a, b, ids, s)
    clipped, norm = ops.clip_grad_norm([da, db], max_norm)
    return h, scores, dh, dx, da, db, clipped, norm


@pytest.mark.parametrize("M,E", [(40, 1), (40, 3), (300, 2)])
def test_a_policy_step(gpu, M, E):
    """All of it as it is used: each part against its formula, and the adapters' gradients against those
    of the whole in 64 bits."""
    announce(f"policy step {M} {E}")
    gen = torch.Generator().manual_seed(M + E)
    H, K, V, r = 256, 128, 3001, 16
    x, w, a, b, ids, s = L.make(gen, M, H, K, E, r, 4, 64, gpu, "mixed")
    head = R.quant(gen, (V,), H, 4, 64, gpu)
    tokens = torch.randint(0, V, (M, 1), generator=gen).int()
    tokens[1] = -1  # a masked place
    tokens = tokens.to(gpu)
    adv = torch.randn(M, 1, generator=gen).to(gpu)
    beta = 0.01
    h, scores, dh, dx, da, db, clipped, norm = policy_step(x, w, a, b, ids, s, head, tokens, adv, beta, 0.1)
    W, HW = R.values(*w, 4, 64), R.values(*head, 4, 64)
    assert torch.equal(check_forward(x, w, a, b, ids, s, 64, 4), h)
    beta32 = torch.full((M,), -beta, device=gpu)
    assert torch.equal(check_logprobs_grad(h, head, HW, tokens, -adv, beta32), dh)
    for p, q in zip(check_grad(x, w, a, b, ids, s, 64, 4, dh), (dx, da, db)):
        assert torch.equal(p, q)
    check_clip([da, db], 0.1, clipped, norm)

    # The whole in 64 bits at the layer's rounded output.
    A64, B64 = (t.double().requires_grad_() for t in (a, b))
    part = torch.zeros(M, H, dtype=torch.float64, device=gpu)
    for e in range(E):
        m = (ids == e).double()[:, None]
        part = part + m * float(s[e]) * ((x.double() @ A64[e].T) @ B64[e].T)
    y = x.double() @ W.T + part
    y = y + (h.double() - y).detach()
    logits = y @ HW.T
    lp = torch.log_softmax(logits, -1)
    given = torch.where(tokens >= 0, lp.gather(1, tokens.clamp(min=0).long()), torch.zeros_like(adv, dtype=torch.float64))
    ent = -(lp.exp() * lp).sum(-1)
    loss = -(adv.double() * given).sum() - float(beta32[0].neg()) * ent.sum()
    ga, gb = torch.autograd.grad(loss, (A64, B64))
    # A logit's gradient is  a [given] - p (A + c (log p + H)):  its terms' magnitudes are size.  It is off
    # by a rounding (half of bf16's step, relative), by p's and log p's errors (el, as the gradient's own
    # test has them) and by H's; dh is the sum of it over the vocabulary's weights, rounded once more.  What
    # is off in dh enters the adapters' gradients through sums of magnitudes.
    ref = Ref(h, HW, tokens, 1.0)
    p, U, half = ref.p, R.U32, R.HALF[torch.bfloat16]
    size = p * (adv.double().abs() + beta * (ref.exact.abs() + ref.H[:, None]))
    size.scatter_add_(1, ref.at, adv.double().abs() * ref.on)
    el = (2 * (ref.el + ref.e_lse))[:, None] + 32 * U * (1 + ref.lse.abs())[:, None]
    ed = size * (2 * half + 4 * el + (V + 128) * U) + p * beta * (2 * el + ref.e_H[:, None])
    ed = ed @ HW.abs()
    # What the products themselves lose (2^-16 of sums of |dh|, which is ed / 2^-7 at most): 2^-7 of ed and
    # more.
    for e in range(E):
        m = ids == e
        X, D, se = x[m].double(), ed[m] * (1 + 2.0 ** -7), abs(float(s[e]))
        R.check(da[e], ga[e], se * (D @ b[e].double().abs()).T @ X.abs() + R.TINY, f"da {e}")
        R.check(db[e], gb[e], se * D.T @ (X.abs() @ a[e].double().abs().T) + R.TINY, f"db {e}")
