"""The norm over many gradients, and the gradients clipped to it."""
import pytest
import torch

import grad_ref as R
from fastmlx_amd import FmxqError, ops
from gpu_util import announce

pytestmark = pytest.mark.gpu


def make(gen, shapes, dtype, dev, scale=1.0):
    """dtype None: both types in turn."""
    t = [dtype or (torch.float32, torch.bfloat16)[i % 2] for i in range(len(shapes))]
    return [(scale * torch.randn(s, generator=gen)).to(d).to(dev) for s, d in zip(shapes, t)]


def check(grads, max_norm, got, norm):
    want = torch.sqrt(sum((g.double() ** 2).sum() for g in grads))
    # Squares and sums in 64 bits: the norm's one rounding to fp32 is all.
    R.check(norm, want, want * R.U32 * 1.001, "norm")
    f = torch.clamp(max_norm / want, max=1.0)
    for i, (g, o) in enumerate(zip(grads, got)):
        ref = g.double() * f
        # The factor to fp32, the product, the type.
        bound = ref.abs() * (3 * R.U32 + (R.HALF[g.dtype] if g.dtype is torch.bfloat16 else 0)) + 1e-44
        assert o.dtype is g.dtype
        R.check(o, ref, bound, f"tensor {i}")


SHAPES = [
    [(1,)], [(7,)], [(64, 128)], [(8192,), (8193,)], [(3, 5, 7), (1,), (4096, 33), (100001,)],
    [(16, 1000), (1000, 16)] * 90, [(5,)] * 333, [(3_000_017,), (12,)],
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, None])
@pytest.mark.parametrize("k", range(len(SHAPES)))
def test_clip(gpu, k, dtype):
    announce(f"clip {k} {dtype}")
    gen = torch.Generator().manual_seed(k)
    grads = make(gen, SHAPES[k], dtype, gpu)
    norm = ops.grad_norm(grads)
    got, same = ops.clip_grad_norm(grads, 0.75)
    assert torch.equal(norm, same) and norm.dim() == 0
    check(grads, 0.75, got, norm)
    # Within the norm: the same bits.
    got, _ = ops.clip_grad_norm(grads, 1e9)
    for g, o in zip(grads, got):
        assert torch.equal(g, o)
    # In place.
    mine = [g.clone() for g in grads]
    again, _ = ops.clip_grad_norm(mine, 0.75, outs=mine)
    check(grads, 0.75, mine, norm)
    assert again is mine


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_any_alignment(gpu, dtype):
    gen = torch.Generator().manual_seed(1)
    flat = make(gen, [(50_000,)], dtype, gpu)[0]
    cuts = [0, 1, 4, 1029, 1030, 20_001, 49_999]
    grads = [flat[a:b] for a, b in zip(cuts, cuts[1:])]
    out = torch.full((50_002,), 9.0, dtype=dtype, device=gpu)
    outs = [out[a + 1:b + 1] for a, b in zip(cuts, cuts[1:])]
    _, norm = ops.clip_grad_norm(grads, 2.0, outs=outs)
    check(grads, 2.0, outs, norm)
    assert out[0] == 9.0 and bool((out[50_000:] == 9.0).all())  # what lies around stays


def test_largest_and_smallest_values(gpu):
    """Squares beyond fp32's range, and below it."""
    for v in (3e38, 1e25, 1e-30, 2e-39):
        grads = [torch.full((1000,), v, device=gpu), torch.full((3,), -v, device=gpu)]
        got, norm = ops.clip_grad_norm(grads, abs(v))
        want = torch.tensor(float(grads[0][0]) * 1003 ** 0.5, dtype=torch.float64, device=gpu)
        if want > 3.4e38:  # the norm has no fp32 value; the scale does
            assert norm.isinf()
        else:
            R.check(norm, want, want * R.U32 * 1.001 + 1e-45, "norm")
        f = float(abs(v) / want)
        ref = grads[0].double() * f
        R.check(got[0], ref, ref.abs() * 3 * R.U32 + 3e-45, "clipped")


def test_no_norm_to_scale_by(gpu):
    for bad in (float("nan"), float("inf")):
        grads = [torch.randn(1000, device=gpu), torch.randn(10, device=gpu).bfloat16()]
        grads[0][17] = bad
        got, norm = ops.clip_grad_norm(grads, 1.0)
        assert norm.isnan() if bad != bad else norm.isinf()
        for g, o in zip(grads, got):
            assert torch.equal(g.nan_to_num(7.0), o.nan_to_num(7.0))
    zeros = [torch.zeros(9, device=gpu)]
    got, norm = ops.clip_grad_norm(zeros, 1.0)
    assert norm == 0 and not got[0].any()
    got, norm = ops.clip_grad_norm([torch.ones(9, device=gpu)], 0.0)
    assert norm == 3 and not got[0].any()


def test_empty_tensors(gpu):
    grads = [torch.empty(0, device=gpu), torch.full((4,), 2.0, device=gpu), torch.empty(0, 3, device=gpu)]
    got, norm = ops.clip_grad_norm(grads, 1.0)
    assert norm == 4 and torch.equal(got[1], torch.full((4,), 0.5, device=gpu))
    assert ops.grad_norm([grads[0]]) == 0


def test_repeats_streams_and_graphs(gpu):
    gen = torch.Generator().manual_seed(2)
    grads = make(gen, [(1000, 37), (513,)] * 100, None, gpu)
    outs = [torch.empty_like(g) for g in grads]
    _, norm = ops.clip_grad_norm(grads, 1.0, outs=outs)
    want = [o.clone() for o in outs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, n = ops.clip_grad_norm(grads, 1.0)
        assert torch.equal(n, norm) and all(torch.equal(p, q) for p, q in zip(got, want))
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _, n = ops.clip_grad_norm(grads, 1.0, outs=outs)
    for k in range(3):
        for g in grads:
            g.mul_(1.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, norm = ops.clip_grad_norm(grads, 1.0)
        assert torch.equal(n, norm), k
        assert all(torch.equal(p, q) for p, q in zip(outs, want)), k


def test_refuses(gpu):
    g = [torch.ones(8, device=gpu), torch.ones(8, device=gpu)]
    with pytest.raises(ValueError):
        ops.grad_norm([])
    with pytest.raises(TypeError):
        ops.grad_norm([g[0].half()])
    with pytest.raises(ValueError):
        ops.grad_norm([g[0], g[1].cpu()])
    with pytest.raises(ValueError):
        ops.grad_norm([torch.ones(4, 4, device=gpu).t()])
    with pytest.raises(ValueError):
        ops.clip_grad_norm(g, 1.0, outs=g[:1])
    with pytest.raises(TypeError):
        ops.clip_grad_norm(g, 1.0, outs=[g[0], g[1].bfloat16()])
    with pytest.raises(ValueError):
        ops.clip_grad_norm(g, 1.0, outs=[g[0], g[1].view(2, 4)])
    for outs in ([g[0], g[0]], [g[1], g[0]]):  # one result twice; another's gradient
        with pytest.raises(FmxqError):
            ops.clip_grad_norm(g, 1.0, outs=outs)
    with pytest.raises(FmxqError):
        ops.clip_grad_norm([g[0], g[0]], 1.0, outs=[g[0], g[0]])
    for bad in (-1.0, float("nan")):
        with pytest.raises(FmxqError):
            ops.clip_grad_norm(g, bad)
    assert all(bool((t == 1).all()) for t in g)
