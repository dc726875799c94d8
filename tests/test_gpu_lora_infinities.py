"""What rows and adapters hold where t = x A^T (or dt = s dy B) leaves bf16's range, or an operand is infinite."""
import pytest
import torch

import lora_ref as L
from fastmlx_amd import ops
from gpu_util import announce
from test_gpu_lora import check_forward, check_grad

pytestmark = pytest.mark.gpu

SIZES = [
    # M, N, K, E, r: few rows, chunks of 64, whole tiles of the wide product, tiles, a panel
    (6, 72, 256, 2, 16), (100, 72, 256, 2, 16), (300, 264, 256, 2, 16), (700, 4104, 512, 3, 72), (1000, 4100, 320, 2, 8),
    (1900, 4102, 320, 2, 16),
]


def make(gpu, M, N, K, E, r, seed=1):
    gen = torch.Generator().manual_seed(seed)
    x, w, a, b, ids, s = L.make(gen, M, N, K, E, r, 4, 64, gpu, "mixed")
    ids[0] = 1
    b = torch.where(b == 0, torch.ones_like(b), b)
    return x, w, a, b, ids, s, torch.randn(M, N, generator=gen).bfloat16().to(gpu)


@pytest.mark.parametrize("M,N,K,E,r", SIZES)
def test_values_between_bf16s_largest_and_fp32s(gpu, M, N, K, E, r):
    """A finite t that bf16 would round to infinity: everything stays finite and right."""
    announce(f"lora large t {M} {N} {K} {E} {r}")
    x, w, a, b, ids, s, dy = make(gpu, M, N, K, E, r)
    big = torch.finfo(torch.bfloat16).max
    # Only one column of x meets the large value, and only one row of it is not zero there.
    x[:, 3] = 0
    x[0] = 0
    x[0, 3] = 1
    a[1, 2, 3] = big
    s[1] = 1.0030  # s t = 3.3997e38: past bf16's last midpoint 3.3962e38, below fp32's 3.4028e38
    b[1, :, 2] = (b[1, :, 2].float() * 1e-33).bfloat16()
    y = check_forward(x, w, a, b, ids, s, 64, 4)
    assert y.isfinite().all()
    # dt: the same through B, in a column of dy.
    x, w, a, b, ids, s, dy = make(gpu, M, N, K, E, r)
    dy[:, 5] = 0
    dy[0] = 0
    dy[0, 5] = 1
    b[1, 5, 2] = big
    s[1] = 1.0030
    a[1, 2] = (a[1, 2].float() * 1e-33).bfloat16()
    x[0] = (x[0].float() * 1e-3).bfloat16()
    g = check_grad(x, w, a, b, ids, s, 64, 4, dy)
    assert all(t.isfinite().all() for t in g)


@pytest.mark.parametrize("M,N,K,E,r", SIZES)
@pytest.mark.parametrize("sign", [1, -1])
def test_an_infinite_t(gpu, M, N, K, E, r, sign):
    """t past fp32's range: infinities of the formula's signs, in that row and in that adapter's gradient."""
    announce(f"lora infinite t {M} {N} {K} {E} {r} {sign}")
    x, w, a, b, ids, s, dy = make(gpu, M, N, K, E, r)
    clean = ops.quantized_matmul_lora(x, *w, a, b, ids, s)
    gclean = ops.quantized_matmul_lora_grad(dy, x, *w, a, b, ids, s)
    x2 = x.clone()
    x2[:, 3] = 0
    base = ops.quantized_matmul_lora(x2, *w, a, b, ids, s)
    x2[0, 3] = 4
    a2 = a.clone()
    a2[1, 2, 3] = sign * 3e38
    y = ops.quantized_matmul_lora(x2, *w, a2, b, ids, s)
    inf = torch.full_like(b[1, :, 2].float(), float("inf"))
    assert torch.equal(y[0].float(), torch.copysign(inf, sign * b[1, :, 2].float()))
    assert torch.equal(y[1:], base[1:])
    dx, da, db = ops.quantized_matmul_lora_grad(dy, x2, *w, a2, b, ids, s)
    # db[1][:, 2] = s sum dy t: row 0's t alone is infinite.
    want = torch.copysign(inf, sign * dy[0].float())
    on = dy[0] != 0
    assert torch.equal(db[1, :, 2][on], want[on])
    rest = torch.arange(r, device=gpu) != 2
    assert db[1][:, rest].isfinite().all() and db[0].isfinite().all()
    # dt, through B: rows of dx and that adapter's da.
    dy2 = dy.clone()
    dy2[:, 5] = 0
    dy2[0, 5] = 4
    b2 = b.clone()
    b2[1, 5, 2] = sign * 3e38
    a3 = torch.where(a == 0, torch.ones_like(a), a)
    dx, da, db = ops.quantized_matmul_lora_grad(dy2, x, *w, a3, b2, ids, s)
    infk = torch.full_like(a3[1, 2].float(), float("inf"))
    assert torch.equal(dx[0].float(), torch.copysign(infk, sign * a3[1, 2].float()))
    on = x[0] != 0
    assert torch.equal(da[1, 2][on], torch.copysign(infk, sign * x[0].float())[on])
    assert da[1][rest].isfinite().all() and da[0].isfinite().all()
    assert clean.isfinite().all() and all(t.isfinite().all() for t in gclean)


@pytest.mark.parametrize("M,N,K,E,r", SIZES)
def test_infinite_operands(gpu, M, N, K, E, r):
    """Results are not finite exactly where the formula's are not."""
    announce(f"lora infinite operands {M} {N} {K} {E} {r}")
    x, w, a, b, ids, s, dy = make(gpu, M, N, K, E, r)
    x[0, 3] = float("inf")
    y = ops.quantized_matmul_lora(x, *w, a, b, ids, s)
    assert not y[0].isfinite().any() and y[1:].isfinite().all()
    dx, da, db = ops.quantized_matmul_lora_grad(dy, x, *w, a, b, ids, s)
    col = torch.arange(K, device=gpu) == 3
    assert dx.isfinite().all() and not da[1][:, col].isfinite().any() and da[1][:, ~col].isfinite().all()
    assert not db[1].isfinite().any() and db[0].isfinite().all() and da[0].isfinite().all()
    # An infinity of A reaches its row of t, and of B its output and its column of dt.
    x, w, a, b, ids, s, dy = make(gpu, M, N, K, E, r)
    a[1, 2, 3], mine = float("inf"), ids == 1
    y = ops.quantized_matmul_lora(x, *w, a, b, ids, s)
    assert not y[mine].isfinite().any() and y[~mine].isfinite().all()
    dx, da, db = ops.quantized_matmul_lora_grad(dy, x, *w, a, b, ids, s)
    assert not dx[mine][:, col].isfinite().any() and dx[:, ~col].isfinite().all() and dx[~mine].isfinite().all()
    assert da.isfinite().all() and db[0].isfinite().all()
    assert not db[1][:, 2].isfinite().any() and db[1][:, torch.arange(r, device=gpu) != 2].isfinite().all()
    x, w, a, b, ids, s, dy = make(gpu, M, N, K, E, r)
    b[1, 7, 2] = float("inf")
    y = ops.quantized_matmul_lora(x, *w, a, b, ids, s)
    out = torch.arange(N, device=gpu) == 7
    assert not y[mine][:, out].isfinite().any() and y[:, ~out].isfinite().all() and y[~mine].isfinite().all()
