"""Log probabilities of given tokens, entropy, likeliest tokens and their gradient, against 64-bit
references."""
import pytest
import torch

import grad_ref as R
from fastmlx_amd import FmxqError, ops
from gpu_util import announce

pytestmark = pytest.mark.gpu
U = R.U32


def case(gpu, M, V, K, k, bits=4, group=64, seed=1, scale=1.0, absent=0.1):
    gen = torch.Generator().manual_seed(seed)
    w = R.quant(gen, (V,), K, bits, group, gpu)
    W = R.values(*w, bits, group)
    ids = torch.randint(0, V, (M, k), generator=gen)
    ids[torch.rand(M, k, generator=gen) < absent] = -1
    lean = W[ids[:, 0].clamp(min=0).to(gpu)].cpu() * 2 * torch.rand(M, 1, generator=gen)
    h = (scale * (torch.randn(M, K, generator=gen) + lean)).bfloat16().to(gpu)
    return h, w, W, ids.int().to(gpu), gen


class Ref:
    """The definition in 64 bits, and bounds.  el: a logit's error, an fp32 sum of K products, the scaling
    and constants in fp32.  es: fp32 sums over a tile and over tiles."""

    def __init__(self, h, W, ids, T):
        V, K = W.shape
        self.ids = ids.long()
        self.on = (self.ids >= 0) & (self.ids < V)
        self.at = torch.where(self.on, self.ids, torch.zeros_like(self.ids))
        self.l = h.double() @ W.T / T
        self.lse = torch.logsumexp(self.l, -1)
        self.logp = self.l - self.lse[:, None]
        self.p = self.logp.exp()
        top = self.p.amax(-1)
        at = self.p.argmax(-1)
        # What the likeliest token leaves, summed without it.
        rest = self.p.clone()
        rest.scatter_(1, at[:, None], 0.0)
        left = rest.sum(-1)
        self.first = at
        self.neg_top = torch.log1p(left / top)
        self.H = top * self.neg_top + (rest * -self.logp).sum(-1)
        size = (h.double().abs() @ W.abs().T).amax(-1) / T
        self.el = (K + 16) * U * size
        self.es = (min(V, 2048) + 64) * U
        # Exponentials below fp32's normal range are lost: V of 2^-126 at most, times the distance (126
        # ln 2 < 88, and a little more where several reach it) for the entropy.
        self.lost = V * 2.0 ** -126
        self.rel = 4 * self.el + self.es + 32 * U
        self.e_lse = 2 * self.el + self.es + 16 * U * (1 + self.lse.abs())
        # Of log p: the logit's error and the sum's; of the likeliest token's all relative to it.
        self.e_logp = 3 * self.el[:, None] + self.es + 16 * U * (1 + self.logp.abs())
        self.e_logp.scatter_(1, at[:, None], (self.rel * self.neg_top + self.lost)[:, None])
        # The entropy's terms are positive; each p is off by rel, each log p of the others by 2 el.
        self.e_H = 2 * self.rel * self.H + (2 * self.el + 16 * U) * left + 90 * self.lost
        exact = self.logp.clone()
        exact.scatter_(1, at[:, None], -self.neg_top[:, None])
        self.given = torch.where(self.on, exact.gather(1, self.at), torch.zeros_like(exact[:, :1]))
        self.e_given = torch.where(self.on, self.e_logp.gather(1, self.at), torch.zeros_like(exact[:, :1]))
        self.exact = exact


def check_scores(h, w, W, ids, top, T=1.0, group=64, bits=4):
    got = ops.head_logprobs(h, *w, ids, top=top, temperature=T, group_size=group, bits=bits)
    r = Ref(h, W, ids, T)
    R.check(got[0], r.given, r.e_given + 1e-37, "logp")
    R.check(got[1], r.H, r.e_H + 1e-37, "entropy")
    R.check(got[2], r.lse, r.e_lse, "lse")
    if top:
        want = torch.sort(r.l, dim=-1, descending=True, stable=True).indices[:, :top]
        ti = got[3].long()
        # Logits that differ by less than 64-bit sums do are equal here.
        same = (r.l.gather(1, ti) - r.l.gather(1, want)).abs() <= 1e-13 * r.l.abs().amax(-1, keepdim=True)
        assert bool((same | (ti == want)).all()), "top ids"
        assert all(len(set(row)) == top for row in ti.tolist())
        R.check(got[4], r.exact.gather(1, ti), r.e_logp.gather(1, ti) + 1e-37, "top_logp")
    return got, r


SCORES = [
    # M, V, K, k, top, bits, group, T
    (1, 1000, 64, 1, 5, 4, 64, 1.0), (1, 32000, 512, 1, 20, 4, 64, 1.0), (3, 37, 32, 2, 8, 4, 32, 0.7),
    (17, 5001, 128, 4, 1, 8, 64, 1.0), (33, 3001, 256, 64, 64, 4, 128, 1.3), (64, 2000, 320, 1, 64, 4, 64, 1.0),
    (65, 777, 512, 3, 10, 8, 32, 1.0), (100, 30000, 256, 1, 0, 4, 64, 1.0), (130, 20001, 192, 2, 33, 4, 64, 0.5),
    (300, 1001, 128, 1, 64, 4, 64, 1.0), (509, 12345, 256, 1, 5, 4, 128, 1.0), (700, 300, 64, 1, 3, 8, 64, 1.0),
    (1800, 5003, 128, 2, 20, 4, 64, 1.0), (2049, 3000, 256, 1, 64, 8, 64, 2.0), (1, 1, 64, 1, 1, 4, 64, 1.0),
    (70, 64, 64, 1, 64, 4, 64, 1.0), (5, 2, 64, 1, 2, 4, 64, 1.0),
]


@pytest.mark.parametrize("M,V,K,k,top,bits,group,T", SCORES)
def test_scores(gpu, M, V, K, k, top, bits, group, T):
    announce(f"logprobs {M} {V} {K} {k} {top} {bits} {group} {T}")
    h, w, W, ids, _ = case(gpu, M, V, K, k, bits, group, seed=M + V)
    check_scores(h, w, W, ids, top, T, group, bits)


def test_scores_without_tokens(gpu):
    h, w, W, ids, _ = case(gpu, 20, 900, 64, 1)
    got, _ = check_scores(h, w, W, ids[:, :0].contiguous(), 4)
    assert got[0].shape == (20, 0)


def test_scores_in_chunks_of_rows(gpu):
    """More rows than a chunk's exponentials: 130000 tokens take chunks of 2560."""
    M, V = 3400, 130000
    h, w, W, ids, _ = case(gpu, M, V, 64, 1)
    got = ops.head_logprobs(h, *w, ids, top=3)
    for rows in (slice(0, 40), slice(3300, 3400)):
        part = ops.head_logprobs(h[rows].contiguous(), *w, ids[rows].contiguous(), top=3)
        assert torch.equal(part[3], got[3][rows])
        r = Ref(h[rows], W, ids[rows], 1.0)
        R.check(got[0][rows], r.given, r.e_given + 1e-37, "logp")
        R.check(got[1][rows], r.H, r.e_H + 1e-37, "entropy")
        R.check(got[4][rows], r.exact.gather(1, got[3][rows].long()),
                r.e_logp.gather(1, got[3][rows].long()) + 1e-37, "top_logp")


@pytest.mark.parametrize("M,V", [(20, 3000), (300, 9000), (1800, 3000)])
@pytest.mark.parametrize("scale", [1e-9, 0.02, 8.0, 100.0])
def test_flat_and_sure_rows(gpu, M, V, scale):
    """From all tokens alike to one that takes everything: log p and entropy to their own size."""
    h, w, W, ids, _ = case(gpu, M, V, 128, 2, seed=3, scale=scale)
    _, r = check_scores(h, w, W, ids, 7)
    if scale == 100.0:
        assert float(r.H.min()) < 1e-6


@pytest.mark.parametrize("M", [4, 100, 1800])
def test_equal_logits_go_to_the_lower_token(gpu, M):
    """A vocabulary of few different rows, and rows of zeros."""
    V, K = 5000, 128
    h, w, _, ids, gen = case(gpu, M, V, K, 1)
    pick = torch.randint(0, 40, (V,), generator=gen).to(gpu)
    w = tuple(t[pick].contiguous() for t in w)
    h[1] = 0
    h[M - 1] = 0
    got = ops.head_logprobs(h, *w, ids, top=50)
    few = h.double() @ R.values(*w, 4, 64)[[int((pick == i).nonzero()[0]) for i in range(40)]].T
    l = few[:, pick]  # equal rows have equal logits
    want = torch.sort(l, dim=-1, descending=True, stable=True).indices[:, :50]
    assert torch.equal(got[3].long(), want)
    assert torch.equal(got[3][1].long(), torch.arange(50, device=gpu))
    flat = torch.log(torch.tensor(V, dtype=torch.float64, device=gpu))
    for t in (got[1][1], got[2][1], -got[4][1]):
        R.check(t, flat.expand(t.shape), (flat * 4 * U).expand(t.shape), "flat row")


@pytest.mark.parametrize("M", [10, 90, 1800])
def test_nearly_equal_logits(gpu, M):
    """Logits that differ by less than fp32 sums see: ordered by their exact values."""
    V, K = 4000, 512
    h, w, W, ids, gen = case(gpu, M, V, K, 1)
    # Columns of h that only separate copies of one row by the last bit of a scale.
    words, s, b = (t.clone() for t in w)
    copies = torch.randperm(V, generator=gen)[:60].to(gpu)
    words[copies], s[copies], b[copies] = w[0][0], w[1][0], w[2][0]
    h[:] = W[0].bfloat16() * 0.5
    h[:, :64] *= 1e-4
    s[copies, 0] = s[0, 0] * (1 + 2.0 ** -6 * torch.arange(60, device=gpu)).bfloat16()
    w = (words, s, b)
    W = R.values(*w, 4, 64)
    check_scores(h, w, W, ids, 50)


@pytest.mark.parametrize("M,V", [(20, 3000), (90, 9000), (1800, 3000)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_bad_rows_stay_alone(gpu, M, V, value):
    h, w, W, ids, _ = case(gpu, M, V, 128, 2, absent=0.0)
    clean = ops.head_logprobs(h, *w, ids, top=9)
    h2 = h.clone()
    h2[7, 3] = value
    got = ops.head_logprobs(h2, *w, ids, top=9)
    keep = torch.arange(M, device=gpu) != 7
    for p, q in zip(got, clean):
        assert torch.equal(p[keep], q[keep])
    for i in (0, 1, 2, 4):
        assert got[i][7].isnan().all()
    assert bool((got[3][7] == -1).all())
    a = torch.randn(M, 2, device=gpu)
    d = ops.head_logprobs_grad(h, *w, ids, *clean[:3], a)
    d2 = ops.head_logprobs_grad(h2, *w, ids, *got[:3], a)
    assert torch.equal(d[keep], d2[keep]) and d2[7].isnan().all()
    a[7] = 0  # nothing flows back
    assert not ops.head_logprobs_grad(h2, *w, ids, *got[:3], a)[7].any()


def test_ids_out_of_range_are_absent_and_reported(gpu):
    h, w, W, ids, _ = case(gpu, 12, 500, 64, 3)
    ids[2, 1] = 500
    ids[3, 0] = -2**31
    ops.device_error()
    got, _ = check_scores(h, w, W, ids, 0)
    assert got[0][2, 1] == 0
    with pytest.raises(FmxqError):
        ops.device_error()
    check_grad(h, w, W, ids, torch.ones(12, 3, device=gpu), None)
    with pytest.raises(FmxqError):
        ops.device_error()
    ops.device_error()


# ---- gradient -------------------------------------------------------------------------


def check_grad(h, w, W, ids, a, c, T=1.0, group=64, bits=4):
    form = dict(temperature=T, group_size=group, bits=bits)
    scores = ops.head_logprobs(h, *w, ids, **form)
    dh = ops.head_logprobs_grad(h, *w, ids, *scores, a, grad_entropy=c, **form)
    r = Ref(h, W, ids, T)
    V = W.shape[0]
    on = torch.where(r.on, a.double(), torch.zeros_like(a, dtype=torch.float64))
    A = on.sum(-1, keepdim=True)
    C = (c.double() if c is not None else torch.zeros(len(h), dtype=torch.float64, device=h.device))[:, None]
    lp, p, H = r.exact, r.p, r.H[:, None]
    want = torch.zeros_like(p).scatter_add_(1, r.at, on)
    given = torch.zeros_like(p).scatter_add_(1, r.at, r.on.double()) > 0
    mag = torch.zeros_like(p).scatter_add_(1, r.at, on.abs())
    flow = A + C * (lp + H)
    d = want - p * flow
    # e to bf16 once (not the given tokens'), p and log p by the logits' and lse's errors, H's own.
    el = (2 * (r.el + r.e_lse))[:, None] + 32 * U * (1 + r.lse.abs())[:, None]
    size = p * (A.abs() + on.abs().sum(-1, keepdim=True) + C.abs() * (lp.abs() + H))
    ed = size * (4 * el + 64 * U) + p * C.abs() * (2 * el + r.e_H[:, None]) + mag * (4 * el + 16 * U) * (p + (1 - p))
    half = R.HALF[torch.bfloat16]
    ed = ed + torch.where(given, torch.zeros_like(d), half * (p * flow.abs() + ed))
    dh64 = d @ W / T
    e = (ed @ W.abs() + (V + 64) * U * ((p * flow.abs() + mag) @ W.abs())) / T
    R.check(dh, dh64, e + half * (dh64.abs() + e) + R.TINY, "dh")
    return dh


GRADS = [
    # M, V, K, k, bits, group, T, entropy
    (1, 1000, 64, 1, 4, 64, 1.0, True), (2, 37, 96, 3, 4, 32, 0.7, True), (17, 5001, 128, 4, 8, 64, 1.0, False),
    (37, 3001, 256, 1, 8, 64, 1.0, True), (50, 2000, 320, 64, 4, 64, 1.3, True), (64, 900, 128, 9, 4, 128, 1.0, True),
    (65, 777, 512, 2, 8, 32, 1.0, True), (130, 20001, 192, 2, 4, 64, 0.5, True), (300, 1001, 128, 1, 4, 64, 1.0, False),
    (1000, 5003, 128, 1, 4, 64, 0.7, True), (1100, 9000, 256, 3, 4, 64, 1.0, True), (2049, 3000, 64, 1, 8, 64, 1.0, True),
]


@pytest.mark.parametrize("M,V,K,k,bits,group,T,entropy", GRADS)
def test_grad(gpu, M, V, K, k, bits, group, T, entropy):
    announce(f"logprobs grad {M} {V} {K} {k} {bits} {group} {T} {entropy}")
    h, w, W, ids, gen = case(gpu, M, V, K, k, bits, group, seed=M + V)
    a = torch.randn(M, k, generator=gen).to(gpu)
    c = torch.randn(M, generator=gen).to(gpu) if entropy else None
    check_grad(h, w, W, ids, a, c, T, group, bits)


def test_grad_in_pieces(gpu):
    """A vocabulary of several pieces: the sums go on from piece to piece."""
    h, w, W, ids, gen = case(gpu, 1200, 130000, 64, 2)
    a, c = torch.randn(1200, 2, generator=gen).to(gpu), torch.randn(1200, generator=gen).to(gpu)
    rows = slice(1100, 1200)
    form = ops.head_logprobs(h, *w, ids)
    dh = ops.head_logprobs_grad(h, *w, ids, *form, a, c)
    want = check_grad(h[rows].contiguous(), w, W, ids[rows].contiguous(), a[rows].contiguous(), c[rows].contiguous())
    # Both within the bound of the exact value.
    assert float((dh[rows].float() - want.float()).norm()) <= 2 * 2.0 ** -8 * float(want.float().norm())


def test_grad_of_tokens_named_twice_and_of_all_absent(gpu):
    h, w, W, ids, gen = case(gpu, 40, 600, 128, 6)
    ids[:, 3] = ids[:, 0]
    ids[:, 5] = ids[:, 0]
    ids[4] = -1
    a = torch.randn(40, 6, generator=gen).to(gpu)
    a[5] = 0
    dh = check_grad(h, w, W, ids, a, None)
    assert not dh[4].any() and not dh[5].any()


@pytest.mark.parametrize("scale", [8.0, 100.0])
def test_grad_of_sure_rows(gpu, scale):
    """Where the given token takes nearly everything the gradient is what the others leave."""
    h, w, W, ids, gen = case(gpu, 60, 2000, 128, 1, scale=scale, absent=0.0)
    check_grad(h, w, W, ids, torch.ones(60, 1, device=gpu), None)


def test_grad_is_cross_entropys(gpu):
    """The gradient of -logp of one token is head_cross_entropy's."""
    h, w, W, ids, gen = case(gpu, 70, 3000, 128, 1, absent=0.0)
    loss, lse, dh = ops.head_cross_entropy(h, *w, ids[:, 0].contiguous(), grad=True)
    s = ops.head_logprobs(h, *w, ids)
    mine = ops.head_logprobs_grad(h, *w, ids, *s, torch.full((70, 1), -1.0, device=gpu))
    r = Ref(h, W, ids, 1.0)
    R.check(s[0][:, 0], -loss.double(), 2 * r.e_given[:, 0] + 64 * U * loss.double(), "logp")
    scale = (r.p @ W.abs()) + W[ids[:, 0].long()].abs()
    R.check(mine, dh.double(), 2.0 ** -6 * scale, "dh")


def test_grad_against_differences(gpu):
    h, w, W, ids, gen = case(gpu, 4, 50, 64, 2, scale=0.3, absent=0.0)
    a, c = torch.randn(4, 2, generator=gen), torch.randn(4, generator=gen)

    def loss(x):
        lp = torch.log_softmax(x @ W.cpu().T / 0.8, -1)
        return (lp.gather(1, ids.cpu().long()) * a).sum() - (c[:, None] * lp.exp() * lp).sum()

    s = ops.head_logprobs(h, *w, ids, temperature=0.8)
    dh = ops.head_logprobs_grad(h, *w, ids, *s, a.to(gpu), c.to(gpu), temperature=0.8).double().cpu()
    x = h.double().cpu()
    d = torch.randn(x.shape, generator=gen, dtype=torch.float64)
    slope = (loss(x + 1e-6 * d) - loss(x - 1e-6 * d)) / 2e-6
    # bf16 twice: the coefficients and the result.
    assert abs(float((dh * d).sum() - slope)) <= 2.0 ** -7 * float((dh.abs() * d.abs()).sum()) + 1e-3


def run_all(c):
    h, w, ids, a, e = c
    s = ops.head_logprobs(h, *w, ids, top=6)
    return [*s, ops.head_logprobs_grad(h, *w, ids, *s[:3], a, e)]


@pytest.mark.parametrize("M,V", [(9, 5000), (200, 5000), (1900, 2000)])
def test_streams_and_graphs(gpu, M, V):
    h, w, W, ids, gen = case(gpu, M, V, 128, 2)
    c = (h, w, ids, torch.randn(M, 2, generator=gen).to(gpu), torch.randn(M, generator=gen).to(gpu))
    want = run_all(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(p, q) for p, q in zip(run_all(c), want))
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = run_all(c)
    for k in range(3):
        h.copy_(torch.randn(h.shape, generator=gen).bfloat16())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, run_all(c))), k


def test_refuses(gpu):
    h, w, W, ids, _ = case(gpu, 4, 100, 64, 2)
    f = ops.head_logprobs
    with pytest.raises(ValueError):
        f(h, *w, ids[:3])
    with pytest.raises(ValueError):
        f(h, *w, ids[:, 0])
    with pytest.raises(TypeError):
        f(h, *w, ids.long())
    with pytest.raises(ValueError):
        f(h, *w, ids.cpu())
    for top in (-1, 65, 101, 2**40):
        with pytest.raises(FmxqError):
            f(h, *w, ids, top=top)
    with pytest.raises(FmxqError):
        f(h, *w, ids, temperature=0.0)
    with pytest.raises(FmxqError):
        f(h, *w, torch.zeros(4, 65, dtype=torch.int32, device=gpu))
    s = f(h, *w, ids)
    a = torch.ones(4, 2, device=gpu)
    with pytest.raises(ValueError):
        ops.head_logprobs_grad(h, *w, ids, *s, a[:, :1].contiguous())
    with pytest.raises(TypeError):
        ops.head_logprobs_grad(h, *w, ids, *s, a.double())
    with pytest.raises(ValueError):
        ops.head_logprobs_grad(h, *w, ids, *s, a, grad_entropy=a)
    none = torch.zeros(4, 0, device=gpu)
    with pytest.raises(FmxqError):
        ops.head_logprobs_grad(h, *w, ids[:, :0].contiguous(), none, s[1], s[2], none)
    assert [t.shape[0] for t in f(h[:0], *w, ids[:0], top=3)] == [0] * 5


@pytest.mark.parametrize("M,V,K", [(3, 3001, 256), (16, 40000, 1024), (50, 3001, 128), (300, 9000, 128), (1900, 3001, 128)])
def test_a_dirty_workspace(gpu, M, V, K):
    """What a workspace held before makes no difference, and nothing is written behind it."""
    import ctypes

    from fastmlx_amd._lib import load

    announce(f"logprobs dirty workspace {M} {V} {K}")
    lib = load()
    h, w, W, ids, gen = case(gpu, M, V, K, 2)
    a, c = torch.randn(M, 2, generator=gen).to(gpu), torch.randn(M, generator=gen).to(gpu)
    want = ops.head_logprobs(h, *w, ids, top=7)
    dh = ops.head_logprobs_grad(h, *w, ids, *want[:3], a, grad_entropy=c)
    size = ctypes.c_size_t()
    head = [t.data_ptr() for t in (h, *w, ids)]
    st = torch.cuda.current_stream().cuda_stream
    for fill in (0xFF, 0x01):
        got = [torch.empty_like(t) for t in want]
        assert lib.fmxq_head_logprobs_workspace(M, V, K, 2, 7, ctypes.byref(size)) == 0
        ws = torch.full((size.value + 16,), fill, dtype=torch.uint8, device=gpu)
        assert lib.fmxq_head_logprobs(*head, *(t.data_ptr() for t in got), M, V, K, 2, 7, 1.0, 64, 4, ws.data_ptr(),
                                      size.value, st) == 0
        assert bool((ws[size.value:] == fill).all())
        for p, q in zip(got, want):
            assert torch.equal(p, q)
        assert lib.fmxq_head_logprobs_grad_workspace(M, V, K, 2, ctypes.byref(size)) == 0
        ws = torch.full((size.value + 16,), fill, dtype=torch.uint8, device=gpu)
        out = torch.empty_like(dh)
        assert lib.fmxq_head_logprobs_grad(*head, *(t.data_ptr() for t in want[:3]), a.data_ptr(), c.data_ptr(),
                                           out.data_ptr(), M, V, K, 2, 1.0, 64, 4, ws.data_ptr(), size.value, st) == 0
        assert bool((ws[size.value:] == fill).all())
        assert torch.equal(out, dh)
