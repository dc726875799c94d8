"""Losses of a quantized head and input gradients of the quantized products, on the GPU,
against 64-bit references with derived bounds (tests/grad_ref.py)."""
import pytest
import torch

import grad_ref as ref
from fastmlx_amd import FmxqError, ops
from gpu_util import announce

pytestmark = pytest.mark.gpu


def hidden(gen, M, K, dev, scale=1.0):
    return (scale * torch.randn(M, K, generator=gen)).bfloat16().to(dev)


def ce_case(gpu, M, V, K, bits=4, group=64, seed=1, scale=1.0, ignored=0.1):
    gen = torch.Generator().manual_seed(seed)
    w = ref.quant(gen, (V,), K, bits, group, gpu)
    h = hidden(gen, M, K, gpu, scale)
    y = torch.randint(0, V, (M,), generator=gen).int().to(gpu)
    if M > 1:
        y[torch.rand(M, generator=gen).to(gpu) < ignored] = -100
    g = torch.rand(M, generator=gen).to(gpu)
    return h, w, y, g


def ce_check(h, w, y, g, bits, group, ignore=-100):
    W = ref.values(*w, bits, group)
    keep = (y >= 0) & (y < W.shape[0]) & (y != ignore)
    ids = torch.where(keep, y, torch.zeros_like(y)).long()[:, None]
    want = ref.head(h, W, ids, keep.double()[:, None], keep, 1.0, g)
    got = ops.head_cross_entropy(h, *w, y, ignore_index=ignore, grad=True, grad_loss=g,
                                 group_size=group, bits=bits)
    only = ops.head_cross_entropy(h, *w, y, ignore_index=ignore, group_size=group, bits=bits)
    for name, a, (r, e) in zip(("loss", "lse", "dh"), got, want):
        ref.check(a, r, e, name)
    for name, a, (r, e) in zip(("loss", "lse"), only, want):
        ref.check(a, r, e, name + " alone")
    return got


CE = [(1, 1, 32, 4, 32), (1, 1000, 64, 4, 64), (2, 7, 96, 8, 32), (5, 255, 128, 4, 128),
      (31, 256, 512, 4, 64), (33, 257, 1056, 4, 32), (64, 4099, 256, 8, 64), (65, 300, 192, 4, 64),
      (130, 1025, 384, 8, 128), (300, 2000, 512, 4, 64), (16, 50257, 128, 4, 64),
      (513, 700, 96, 4, 32), (257, 8192, 1024, 8, 64),
      # tiles of 128 and 256 rows, with part-full last steps, tiles and tokens
      (100, 40000, 256, 4, 128), (70, 60001, 96, 8, 32), (300, 20000, 96, 4, 32),
      (200, 30001, 192, 8, 64), (1000, 9001, 160, 4, 32), (1024, 12800, 320, 4, 64),
      # panels, the last step of 32 values, widths below a tile
      (1100, 24001, 96, 4, 32), (1300, 20001, 320, 8, 64), (2050, 10240, 1056, 4, 32),
      # the logits alone on panels too, and gradients in the lowest tiles
      (2900, 14001, 96, 8, 32), (50, 12345, 1056, 8, 32), (64, 30000, 256, 4, 64)]


@pytest.mark.parametrize("M,V,K,bits,group", CE)
def test_cross_entropy(gpu, M, V, K, bits, group):
    announce(f"ce {M}x{V}x{K} {bits} bits, groups of {group}")
    h, w, y, g = ce_case(gpu, M, V, K, bits, group, seed=M + V)
    ce_check(h, w, y, g, bits, group)
    ops.device_error()


def test_cross_entropy_in_pieces(gpu):
    """Enough rows that the vocabulary is walked in several pieces, the last a short one."""
    announce("ce 66000x4100x64")
    h, w, y, g = ce_case(gpu, 66000, 4100, 64)
    ce_check(h, w, y, g, 4, 64)


@pytest.mark.parametrize("scale", [30.0, 1e-3])
def test_cross_entropy_wide_and_flat_logits(gpu, scale):
    """Logits of hundreds (one token takes everything, tiles far below the row's largest
    underflow) and logits that hardly differ."""
    announce(f"ce scale {scale}")
    h, w, y, g = ce_case(gpu, 40, 1500, 512, scale=scale)
    ce_check(h, w, y, g, 4, 64)


@pytest.mark.parametrize("M,V", [(60, 3000), (150, 30000), (1100, 12000)])
def test_cross_entropy_tiles_of_different_exponents(gpu, M, V):
    """Rows whose largest logits lie within and beyond +-32 and +-96 units of log 2, so that the
    statistics of a row's tiles are relative to one power of two, two, or several."""
    announce(f"ce exponents {M}x{V}")
    h, w, y, g = ce_case(gpu, M, V, 256)
    h = (h * torch.linspace(0.5, 40, M, device=gpu)[:, None]).bfloat16()
    W = ref.values(*w, 4, 64)
    top = (h.double() @ W.double().t()).amax(1) / 0.6931471805599453
    assert top.min() < 28 and top.max() > 100
    ce_check(h, w, y, g, 4, 64)


@pytest.mark.parametrize("M,V", [(12, 900), (150, 30000), (1100, 12000)])
def test_logits_beyond_the_exponents_range(gpu, M, V):
    """Logits of 1e9 and more, whose roundings are larger than any exponent of a power of two:
    one token takes everything and the loss is a difference of logits."""
    announce(f"ce huge logits {M}x{V}")
    h, w, y, g = ce_case(gpu, M, V, 256)
    h = (h * torch.logspace(8, 24, M, device=gpu)[:, None]).bfloat16()
    got = ce_check(h, w, y, g, 4, 64)
    assert all(torch.isfinite(t).all() for t in got)
    ids, t = y.clamp(min=0)[:, None], torch.zeros(M, 1, device=gpu)
    got = ops.head_distill((h * 0 + 1).bfloat16(), *w, ids, t, temperature=1e-10, grad=True)
    assert all(torch.isfinite(t).all() for t in got)


def test_cross_entropy_confident_rows(gpu):
    """Targets that the head is sure of: p - 1 is a small difference of near equals."""
    announce("ce confident")
    h, w, y, g = ce_case(gpu, 24, 900, 512, ignored=0.0)
    W = ref.values(*w, 4, 64)
    h = (W[y.long()] * torch.linspace(1, 30, 24, device=gpu)[:, None]).bfloat16()
    ce_check(h, w, y, g, 4, 64)


def test_cross_entropy_all_ignored_and_bad_targets(gpu):
    announce("ce ignored")
    h, w, y, g = ce_case(gpu, 9, 300, 64)
    loss, lse, dh = ops.head_cross_entropy(h, *w, torch.full_like(y, 7), ignore_index=7, grad=True)
    assert not loss.any() and not dh.any() and torch.isfinite(lse).all()
    ops.device_error()
    y = torch.tensor([0, 299, 300, -1, -100, 5, 2**31 - 1, -2**31, 8], dtype=torch.int32, device=gpu)
    got = ce_check(h, w, y, g, 4, 64)
    assert got[0][2] == 0 and got[0][3] == 0 and not got[2][2].any() and not got[2][6:8].any()
    with pytest.raises(FmxqError, match="INDEX"):
        ops.device_error()


def test_cross_entropy_ignore_index_inside_the_vocabulary(gpu):
    announce("ce ignore 3")
    h, w, y, g = ce_case(gpu, 12, 50, 64, ignored=0.0)
    y[:6] = 3
    ce_check(h, w, y, g, 4, 64, ignore=3)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("M,V", [(20, 600), (70, 600), (90, 50000), (300, 20000), (1100, 20000)])
def test_cross_entropy_bad_row_stays_alone(gpu, value, M, V):
    announce(f"ce row of {value}, {M}x{V}")
    h, w, y, g = ce_case(gpu, M, V, 96, 4, 32, ignored=0.0)
    want = ops.head_cross_entropy(h, *w, y, grad=True, group_size=32)
    h2 = h.clone()
    h2[13, 5] = value
    got = ops.head_cross_entropy(h2, *w, y, grad=True, group_size=32)
    rest = torch.arange(M, device=gpu) != 13
    for a, b in zip(got, want):
        assert torch.equal(a[rest], b[rest])
        assert not torch.isfinite(a[13]).all()


@pytest.mark.parametrize("off", [0, 1, 2])
@pytest.mark.parametrize("M,V,K,bits,group", [
    (3, 100, 192, 4, 32), (20, 300, 384, 8, 64), (1, 70, 640, 4, 128), (40, 700, 576, 4, 32),
    (9, 500, 896, 8, 128), (64, 99, 1152, 4, 64)])
def test_cross_entropy_rows_of_few_groups(gpu, M, V, K, bits, group, off):
    """5 to 18 groups a row, never a multiple of 4, and scales that begin in the middle of
    a 4-byte word."""
    announce(f"ce {M}x{V}x{K} {bits} bits, groups of {group}, scales from {off}")
    h, (w, s, b), y, g = ce_case(gpu, M, V, K, bits, group, seed=M + K)

    def moved(t):
        buf = torch.empty(t.numel() + off, dtype=t.dtype, device=gpu)
        return buf[off:].copy_(t.flatten()).view(t.shape)

    ce_check(h, (w, moved(s), moved(b)), y, g, bits, group)


def test_cross_entropy_bad_last_row_stays_alone(gpu):
    """The rows that a tile has past the last one read the last one's values."""
    announce("ce last row of nan, 5x600")
    h, w, y, g = ce_case(gpu, 5, 600, 96, 4, 32, ignored=0.0)
    want = ops.head_cross_entropy(h, *w, y, grad=True, group_size=32)
    h[4] = float("nan")
    got = ops.head_cross_entropy(h, *w, y, grad=True, group_size=32)
    for a, b in zip(got, want):
        assert torch.equal(a[:4], b[:4]) and torch.isnan(a[4]).all()


def distill_case(gpu, M, V, K, k, bits, group, seed, dtype):
    gen = torch.Generator().manual_seed(seed)
    w = ref.quant(gen, (V,), K, bits, group, gpu)
    h = hidden(gen, M, K, gpu)
    ids = torch.randint(-1 if k > 1 else 0, V, (M, k), generator=gen).int().to(gpu)
    t = (4 * torch.randn(M, k, generator=gen)).to(dtype).to(gpu)
    g = torch.rand(M, generator=gen).to(gpu)
    return h, w, ids, t, g


def distill_check(h, w, ids, t, g, T, bits, group):
    W = ref.values(*w, bits, group)
    at, q, keep = ref.teacher_q(ids, t, W.shape[0], T)
    want = ref.head(h, W, at, q, keep, T, g)
    got = ops.head_distill(h, *w, ids, t, temperature=T, grad=True, grad_loss=g, group_size=group,
                           bits=bits)
    only = ops.head_distill(h, *w, ids, t, temperature=T, group_size=group, bits=bits)
    for name, a, (r, e) in zip(("loss", "lse", "dh"), got, want):
        ref.check(a, r, e, name)
    for name, a, (r, e) in zip(("loss", "lse"), only, want):
        ref.check(a, r, e, name + " alone")
    return got


@pytest.mark.parametrize("M,V,K,k,bits,group,T,dtype", [
    (1, 40, 64, 1, 4, 64, 1.0, torch.float32), (3, 1000, 128, 5, 4, 64, 2.0, torch.bfloat16),
    (33, 257, 96, 20, 8, 32, 0.5, torch.float32), (70, 5000, 512, 64, 4, 128, 1.0, torch.bfloat16),
    (200, 999, 256, 63, 8, 64, 3.0, torch.float32), (18, 50, 64, 64, 4, 32, 1.0, torch.bfloat16)])
def test_distill(gpu, M, V, K, k, bits, group, T, dtype):
    """Ids repeat within a row where k nears V, and some entries are absent."""
    announce(f"distill {M}x{V}x{K} k {k}")
    h, w, ids, t, g = distill_case(gpu, M, V, K, k, bits, group, M + k, dtype)
    distill_check(h, w, ids, t, g, T, bits, group)
    ops.device_error()


def test_distill_rows_without_entries(gpu):
    announce("distill empty rows")
    h, w, ids, t, g = distill_case(gpu, 8, 300, 128, 6, 4, 64, 3, torch.float32)
    ids[2] = -1
    t[3] = float("-inf")
    t[4, 1:] = float("-inf")
    t[5, 0] = torch.finfo(torch.float32).min
    ids[6] = ids[6, 0].clamp(min=0)
    loss, _, dh = distill_check(h, w, ids, t, g, 1.0, 4, 64)
    assert loss[2] == 0 and loss[3] == 0 and not dh[2:4].any()
    ops.device_error()
    ids[1, 2] = 300
    distill_check(h, w, ids, t, g, 1.0, 4, 64)
    with pytest.raises(FmxqError, match="INDEX"):
        ops.device_error()


def test_distill_of_one_sure_entry_is_cross_entropy(gpu):
    announce("distill k 1")
    h, w, y, g = ce_case(gpu, 50, 700, 128, ignored=0.0)
    a = ops.head_cross_entropy(h, *w, y, grad=True, grad_loss=g)
    b = ops.head_distill(h, *w, y[:, None].contiguous(), torch.zeros(50, 1, device=gpu), grad=True,
                         grad_loss=g)
    for u, v in zip(a, b):
        assert torch.equal(u, v)


def test_losses_against_differences(gpu):
    """loss(h + d) - loss(h - d) against dh . 2 d.  The loss is a cumulant function of the logits
    along d: its third derivative is at most R^3 / (6 sqrt 3), R the range of the logits' change."""
    announce("differences")
    h, w, ids, t, g = distill_case(gpu, 32, 400, 128, 4, 4, 64, 5, torch.float32)
    W = ref.values(*w, 4, 64)
    gen = torch.Generator().manual_seed(9)
    d = (torch.randn(32, 128, generator=gen) / 64).to(gpu)
    hi, lo = (h.float() + d).bfloat16(), (h.float() - d).bfloat16()
    at, q, keep = ref.teacher_q(ids, t, 400, 1.0)
    step = (hi.double() - lo.double()) / 2
    mid = ((hi.double() + lo.double()) / 2)
    change = step @ W.T
    third = (change.amax(-1) - change.amin(-1)) ** 3 / (6 * 3 ** 0.5)
    one = torch.ones_like(g)
    # The gradient at the midpoint of the two inputs, which need not be a bf16 value: h's
    # differs from it by its own rounding, whose effect the second derivative bounds.
    h = mid.bfloat16()
    (_, eu), _, (_, ed) = ref.head(h, W, at, q, keep, 1.0, one)
    second = (change.amax(-1) - change.amin(-1)) * \
        (((mid - h.double()) @ W.T).amax(-1) - ((mid - h.double()) @ W.T).amin(-1))
    up = ops.head_distill(hi, *w, ids, t)[0].double()
    down = ops.head_distill(lo, *w, ids, t)[0].double()
    dh = ops.head_distill(h, *w, ids, t, grad=True)[2].double()
    slope = 2 * (dh * step).sum(-1)
    bound = third / 3 + second + 2 * (ed * step.abs()).sum(-1) + 4 * eu
    assert ((up - down - slope).abs() <= bound).all()
    assert bound.mean() < 0.2 * slope.abs().mean()  # the bound says something


@pytest.mark.parametrize("M,N,K,bits,group", [
    (1, 1, 32, 4, 32), (1, 4096, 512, 4, 64), (3, 7, 96, 8, 32), (32, 64, 128, 4, 128),
    (33, 1000, 320, 4, 64), (64, 2048, 1056, 4, 32), (65, 129, 256, 8, 128), (200, 512, 2048, 8, 64),
    (129, 4100, 704, 4, 64), (515, 72, 96, 4, 32), (256, 11008, 256, 4, 64),
    (1000, 333, 1056, 8, 32), (700, 2000, 64, 8, 64),
    # panels
    (1025, 37, 96, 4, 32), (1030, 300, 1056, 8, 32), (2001, 129, 320, 4, 64), (1500, 5000, 256, 4, 128),
    (1026, 64, 2048, 8, 64)])
def test_quantized_matmul_grad(gpu, M, N, K, bits, group):
    announce(f"grad {M}x{N}x{K} {bits} bits, groups of {group}")
    gen = torch.Generator().manual_seed(M + N)
    w = ref.quant(gen, (N,), K, bits, group, gpu)
    dy = hidden(gen, M, N, gpu)
    ref.check(ops.quantized_matmul_grad(dy, *w, group, bits),
              *ref.product(dy, ref.values(*w, bits, group)), "dx")


@pytest.mark.parametrize("M", [2, 66])
def test_quantized_matmul_grad_of_the_widest_rows(gpu, M):
    """2^22 - 8 values a row: 64 and 256 rows of dy end just below 2^29 and 2^31 bytes."""
    N = (1 << 22) - 8
    announce(f"grad {M}x{N}x32")
    gen = torch.Generator().manual_seed(M)
    w = ref.quant(gen, (N,), 32, 4, 32, gpu)
    dy = torch.zeros(M, N, device=gpu, dtype=torch.bfloat16)
    dy[:, -5000:] = torch.randn(M, 5000, generator=gen).bfloat16().to(gpu)
    dy[:, :700] = torch.randn(M, 700, generator=gen).bfloat16().to(gpu)
    at = torch.cat([torch.arange(700), torch.arange(N - 5000, N)]).to(gpu)
    y, e = ref.product(dy[:, at], ref.values(w[0][at], w[1][at], w[2][at], 4, 32))
    ref.check(ops.quantized_matmul_grad(dy, *w, 32, 4), y, e, "dx")


def test_quantized_matmul_grad_takes_batches_and_any_alignment(gpu):
    announce("grad shapes")
    gen = torch.Generator().manual_seed(4)
    w = ref.quant(gen, (72,), 128, 4, 64, gpu)
    W = ref.values(*w, 4, 64)
    dy = hidden(gen, 30, 72, gpu)
    y = ops.quantized_matmul_grad(dy.view(2, 3, 5, 72), *w)
    assert y.shape == (2, 3, 5, 128)
    ref.check(y.view(30, 128), *ref.product(dy, W), "batched")
    odd = torch.empty(30 * 72 + 3, dtype=torch.bfloat16, device=gpu)[3:].view(30, 72)
    odd.copy_(dy)
    assert torch.equal(ops.quantized_matmul_grad(odd, *w), y.view(30, 128))
    assert ops.quantized_matmul_grad(dy[:0], *w).shape == (0, 128)
    assert ops.quantized_matmul_grad(dy[0], *w).shape == (128,)
    none = tuple(t[:0] for t in w)
    assert not ops.quantized_matmul_grad(dy[:, :0].contiguous(), *none).any()


def test_quantized_matmul_grad_bad_rows_stay_alone(gpu):
    """A NaN row of dy, and a weight row with an infinite scale against zeros of dy's padding."""
    announce("grad NaN")
    gen = torch.Generator().manual_seed(6)
    w = ref.quant(gen, (37,), 128, 4, 64, gpu)
    dy = hidden(gen, 40, 37, gpu)
    want = ops.quantized_matmul_grad(dy, *w)
    dy[7, 3] = float("nan")
    got = ops.quantized_matmul_grad(dy, *w)
    rest = torch.arange(40, device=gpu) != 7
    assert torch.equal(got[rest], want[rest]) and torch.isnan(got[7]).all()


@pytest.mark.parametrize("counts,N,K,bits,group", [
    ([1], 8, 32, 4, 32), ([0, 5, 0, 40, 1], 100, 192, 4, 64), ([33] * 7, 64, 1056, 8, 32),
    ([200, 0, 0, 130], 512, 384, 4, 128), ([3] * 70, 37, 128, 8, 64), ([0, 0, 900], 256, 512, 4, 64),
    ([700, 300, 0, 513], 130, 1056, 8, 32), ([256, 257], 72, 320, 4, 64), ([1, 0, 2] * 230, 40, 64, 4, 64),
    ([50, 0, 61, 64], 1000, 96, 4, 32)])
def test_gather_qmm_grad(gpu, counts, N, K, bits, group):
    announce(f"gather grad {len(counts)} experts {N}x{K}")
    gen = torch.Generator().manual_seed(N)
    E, S = len(counts), sum(counts)
    w = ref.quant(gen, (E, N), K, bits, group, gpu)
    W = ref.values(*w, bits, group)
    tail = 5  # rows of no expert
    dy = hidden(gen, S + tail, N, gpu)
    ends = torch.tensor([0] + counts).cumsum(0)
    dx = ops.gather_qmm_grad(dy, *w, ends.int().to(gpu), group, bits)
    for e in range(E):
        a, b = int(ends[e]), int(ends[e + 1])
        ref.check(dx[a:b], *ref.product(dy[a:b], W[e]), f"expert {e}")
    assert not dx[S:].any()
    ops.device_error()


def test_gather_qmm_grad_refuses_bad_offsets(gpu):
    announce("gather grad offsets")
    gen = torch.Generator().manual_seed(8)
    w = ref.quant(gen, (3, 16), 64, 4, 64, gpu)
    dy = hidden(gen, 20, 16, gpu)
    for bad in ([0, 12, 8, 20], [0, 5, 9, 21], [-1, 5, 9, 20]):
        dx = ops.gather_qmm_grad(dy, *w, torch.tensor(bad, dtype=torch.int32, device=gpu))
        assert not dx.any()
        with pytest.raises(FmxqError, match="INDEX"):
            ops.device_error()
    dx = ops.gather_qmm_grad(dy, *w, torch.tensor([4, 4, 9, 11], dtype=torch.int32, device=gpu))
    assert not dx[:4].any() and not dx[11:].any() and dx[4:11].any(-1).all()
    dx = ops.gather_qmm_grad(dy, *w, torch.zeros(4, dtype=torch.int32, device=gpu))
    assert not dx.any()
    ops.device_error()


@pytest.mark.parametrize("M,N", [(40, 37), (100, 500), (300, 72), (1100, 130)])
def test_quantized_matmul_grad_bad_row_stays_alone(gpu, M, N):
    announce(f"grad NaN row, {M}x{N}")
    gen = torch.Generator().manual_seed(M)
    w = ref.quant(gen, (N,), 160, 4, 32, gpu)
    dy = hidden(gen, M, N, gpu)
    want = ops.quantized_matmul_grad(dy, *w, 32)
    dy[17, N - 1] = float("inf")
    got = ops.quantized_matmul_grad(dy, *w, 32)
    rest = torch.arange(M, device=gpu) != 17
    assert torch.equal(got[rest], want[rest]) and not torch.isfinite(got[17]).any()


def test_results_do_not_depend_on_what_the_workspace_held(gpu):
    """Workspaces come with whatever was there: the memory is filled with NaN before each call."""
    announce("dirty workspaces")
    for M, V, K, group in ((3, 70, 96, 32), (40, 300, 128, 64), (100, 3000, 96, 32), (300, 20001, 96, 32),
                           (1100, 7001, 96, 32)):
        h, w, y, g = ce_case(gpu, M, V, K, 4, group, seed=M)
        dy = hidden(torch.Generator().manual_seed(M), M, V, gpu)
        off = torch.tensor([0, M // 3, M], dtype=torch.int32, device=gpu)
        two = tuple(torch.stack([t, t]) for t in w)
        first = None
        for fill in (0, 0xFF):
            junk = [torch.full((n,), fill, dtype=torch.uint8, device=gpu)
                    for n in (1 << 28, 1 << 26, 1 << 22, 1 << 18, 4096, 512)]
            torch.cuda.synchronize()
            del junk
            got = [*ops.head_cross_entropy(h, *w, y, grad=True, group_size=group),
                   *ops.head_cross_entropy(h, *w, y, group_size=group),
                   ops.quantized_matmul_grad(dy, *w, group), ops.gather_qmm_grad(dy, *two, off, group)]
            assert all(torch.isfinite(t).all() for t in got)
            first = first or got
            assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_refuses_strides_and_other_shapes(gpu):
    h, w, y, g = ce_case(gpu, 8, 64, 64)
    with pytest.raises(ValueError, match="contiguous"):
        ops.head_cross_entropy(h.t().contiguous().t(), *w, y)
    with pytest.raises(ValueError, match="shape"):
        ops.head_cross_entropy(h, *w, y[:5].contiguous())
    with pytest.raises(ValueError, match="shape"):
        ops.head_cross_entropy(h, w[0], w[1][:60].contiguous(), w[2], y)
    with pytest.raises(ValueError, match="grad"):
        ops.head_cross_entropy(h, *w, y, grad_loss=g)
    with pytest.raises(TypeError):
        ops.head_cross_entropy(h, *w, y.long())
    with pytest.raises(TypeError):
        ops.head_cross_entropy(h.float(), *w, y)
    with pytest.raises(FmxqError, match="bits"):
        ops.head_cross_entropy(h, *w, y, bits=3)
    with pytest.raises(FmxqError, match="top_k"):
        ops.head_distill(h, *w, y[:, None].expand(8, 65).contiguous(), torch.zeros(8, 65, device=gpu))
    with pytest.raises(ValueError, match="columns"):
        ops.quantized_matmul_grad(h[:, :32].contiguous(), *w)
    with pytest.raises(ValueError, match="shape"):
        ops.gather_qmm_grad(h, *(t[None] for t in w), y[:3].contiguous())


def run_all(c):
    """Every call of a small step, as a list of results."""
    out = list(ops.head_cross_entropy(c["h"], *c["head"], c["y"], grad=True))
    out += ops.head_distill(c["h"], *c["head"], c["ids"], c["t"], temperature=2.0, grad=True)
    out.append(ops.quantized_matmul_grad(out[2], *c["proj"]))
    out += ops.moe_sort(c["h"], c["inds"], 5)
    out.append(ops.gather_qmm_grad(out[-4], *c["experts"], out[-1]))
    return out


def small_step(gpu, seed):
    gen = torch.Generator().manual_seed(seed)
    h = hidden(gen, 21, 128, gpu)
    return dict(h=h, head=ref.quant(gen, (501,), 128, 4, 64, gpu),
                y=torch.randint(0, 501, (21,), generator=gen).int().to(gpu),
                ids=torch.randint(0, 501, (21, 9), generator=gen).int().to(gpu),
                t=torch.randn(21, 9, generator=gen).to(gpu),
                proj=ref.quant(gen, (128,), 256, 4, 64, gpu),
                inds=torch.randint(0, 5, (21, 2), generator=gen).int().to(gpu),
                experts=ref.quant(gen, (5, 128), 192, 4, 64, gpu))


def test_repeats_bit_for_bit_on_streams(gpu):
    announce("streams")
    cases = [small_step(gpu, s) for s in (1, 2)]
    want = [run_all(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run_all(cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_graph_replays(gpu):
    """Two graphs captured on one stream, replayed on two streams at once with eager calls
    between."""
    announce("graphs")
    cases = [small_step(gpu, s) for s in (3, 4)]
    new = [small_step(gpu, s) for s in (5, 6)]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(run_all(c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in cases]
    for turn in range(4):
        want = [run_all(c) for c in cases]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, r in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, r)), turn
        for c, n in zip(cases, new):
            for name in ("h", "y", "ids", "t", "inds"):
                c[name].copy_(n[name] if turn % 2 == 0 else c[name].flip(0))
    ops.device_error()
