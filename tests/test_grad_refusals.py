"""What the training operators refuse, before anything is enqueued (CPU)."""
import ctypes

import pytest
import torch

from fastmlx_amd import _lib, ops

P = 4096  # an aligned address that is never read


def status(name, *args):
    return _lib.STATUS[getattr(_lib.load(), name)(*args)]


def ws(name, *sizes):
    n = ctypes.c_size_t()
    rc = getattr(_lib.load(), name)(*sizes, ctypes.byref(n))
    return _lib.STATUS[rc], n.value


def ce(h=P, w=P, targets=P, gl=None, loss=P, lse=P, dh=P, M=4, V=100, K=64, group=64, bits=4,
       work=P, n=1 << 40):
    return status("fmxq_head_cross_entropy", h, w, P, P, targets, gl, loss, lse, dh, M, V, K, -100,
                  group, bits, work, n, None)


@pytest.mark.parametrize("kw,want", [
    (dict(bits=3), "UNSUPPORTED"), (dict(group=16), "UNSUPPORTED"), (dict(K=65), "SHAPE"),
    (dict(K=0), "SHAPE"), (dict(M=-1), "SHAPE"), (dict(V=-1), "SHAPE"), (dict(V=0), "SHAPE"),
    (dict(M=1 << 25), "SHAPE"), (dict(h=None), "INVALID_ARGUMENT"), (dict(w=None), "INVALID_ARGUMENT"),
    (dict(targets=None), "INVALID_ARGUMENT"), (dict(loss=None), "INVALID_ARGUMENT"),
    (dict(lse=None), "INVALID_ARGUMENT"), (dict(h=P + 2), "INVALID_ARGUMENT"),
    (dict(w=P + 4), "INVALID_ARGUMENT"), (dict(dh=P + 8), "INVALID_ARGUMENT"),
    (dict(dh=None, gl=P), "INVALID_ARGUMENT"), (dict(work=None), "INVALID_ARGUMENT"),
    (dict(work=P + 8), "INVALID_ARGUMENT"), (dict(n=100), "INVALID_ARGUMENT")])
def test_cross_entropy_refuses(kw, want):
    assert ce(**kw) == "FMXQ_ERR_" + want


def distill(ids=P, teacher=P, tb=1, k=4, T=1.0, M=4, n=1 << 40):
    return status("fmxq_head_distill", P, P, P, P, ids, teacher, tb, None, P, P, P, M, 100, 64, k, T,
                  64, 4, P, n, None)


@pytest.mark.parametrize("kw,want", [
    (dict(k=0), "SHAPE"), (dict(k=65), "SHAPE"), (dict(T=0.0), "INVALID_ARGUMENT"),
    (dict(T=-1.0), "INVALID_ARGUMENT"), (dict(T=float("nan")), "INVALID_ARGUMENT"),
    (dict(T=float("inf")), "INVALID_ARGUMENT"), (dict(ids=None), "INVALID_ARGUMENT"),
    (dict(teacher=None), "INVALID_ARGUMENT"), (dict(teacher=P + 2, tb=0), "INVALID_ARGUMENT"),
    (dict(n=0), "INVALID_ARGUMENT")])
def test_distill_refuses(kw, want):
    assert distill(**kw) == "FMXQ_ERR_" + want


def grad(dy=P, w=P, dx=P, M=4, N=16, K=64, group=64, bits=4, work=P, n=1 << 40):
    return status("fmxq_quantized_matmul_grad", dy, w, P, P, dx, M, N, K, group, bits, work, n, None)


def gather(dy=P, off=P, dx=P, S=4, E=3, N=16, K=64, n=1 << 40):
    return status("fmxq_gather_qmm_grad", dy, P, P, P, off, dx, S, E, N, K, 64, 4, P, n, None)


@pytest.mark.parametrize("kw,want", [
    (dict(bits=5), "UNSUPPORTED"), (dict(group=256), "UNSUPPORTED"), (dict(K=96), "SHAPE"),
    (dict(M=-1), "SHAPE"), (dict(N=-1), "SHAPE"), (dict(N=1 << 23), "SHAPE"),
    (dict(dy=None), "INVALID_ARGUMENT"), (dict(w=P + 4), "INVALID_ARGUMENT"),
    (dict(dx=P + 2), "INVALID_ARGUMENT"), (dict(dx=None), "INVALID_ARGUMENT"),
    (dict(work=P + 4), "INVALID_ARGUMENT"), (dict(n=1), "INVALID_ARGUMENT")])
def test_quantized_matmul_grad_refuses(kw, want):
    assert grad(**kw) == "FMXQ_ERR_" + want


def test_widths_past_the_products_offsets_are_refused():
    n = (1 << 22) - 7
    assert grad(N=n) == gather(N=n) == "FMXQ_ERR_SHAPE"
    assert grad(K=1 << 22) == gather(K=1 << 22) == ce(K=1 << 22) == "FMXQ_ERR_SHAPE"


@pytest.mark.parametrize("kw,want", [
    (dict(E=0), "SHAPE"), (dict(E=-1), "SHAPE"), (dict(S=-1), "SHAPE"),
    (dict(off=None), "INVALID_ARGUMENT"), (dict(dy=None), "INVALID_ARGUMENT"),
    (dict(dx=P + 2), "INVALID_ARGUMENT"), (dict(n=1), "INVALID_ARGUMENT")])
def test_gather_qmm_grad_refuses(kw, want):
    assert gather(**kw) == "FMXQ_ERR_" + want


def sort(x=P, inds=P, xs=P, order=P, pos=P, off=P, T=4, k=2, E=8, D=16, n=1 << 40):
    return status("fmxq_moe_sort", x, inds, xs, order, pos, off, T, k, E, D, P, n, None)


@pytest.mark.parametrize("kw,want", [
    (dict(E=0), "UNSUPPORTED"), (dict(E=2049), "UNSUPPORTED"), (dict(k=0), "SHAPE"),
    (dict(T=-1), "SHAPE"), (dict(D=-1), "SHAPE"), (dict(T=1 << 40, k=1 << 40), "SHAPE"),
    (dict(x=None), "INVALID_ARGUMENT"), (dict(inds=P + 2), "INVALID_ARGUMENT"),
    (dict(off=None), "INVALID_ARGUMENT"), (dict(xs=P + 1), "INVALID_ARGUMENT"),
    (dict(n=0), "INVALID_ARGUMENT")])
def test_moe_sort_refuses(kw, want):
    assert sort(**kw) == "FMXQ_ERR_" + want


@pytest.mark.parametrize("name,args", [
    ("fmxq_moe_sort_grad", lambda y, p, o, T, k, D: (y, p, o, T, k, D, None)),
    ("fmxq_moe_unsort", lambda y, p, o, T, k, D: (y, p, P, 0, o, T, k, D, None)),
    ("fmxq_moe_unsort_grad", lambda y, p, o, T, k, D: (P, y, p, P, 1, o, P, T, k, D, None))])
def test_rows_refuse(name, args):
    def call(y=P, p=P, o=P, T=4, k=2, D=16):
        return status(name, *args(y, p, o, T, k, D))

    for kw in (dict(T=-1), dict(k=0), dict(D=-1), dict(T=1 << 31, k=2)):
        assert call(**kw) == "FMXQ_ERR_SHAPE"
    for kw in (dict(y=None), dict(p=None), dict(o=None), dict(p=P + 2), dict(y=P + 1)):
        assert call(**kw) == "FMXQ_ERR_INVALID_ARGUMENT"
    assert call(T=0) == "FMXQ_OK"


def test_workspace_sizes():
    assert ws("fmxq_head_workspace", 0, 100, 64, 1, True) == ("FMXQ_OK", 0)
    small = ws("fmxq_head_workspace", 16, 1000, 64, 1, False)
    large = ws("fmxq_head_workspace", 16, 1000, 64, 1, True)
    assert small[0] == large[0] == "FMXQ_OK" and 0 < small[1] < large[1]
    # The logits of a large batch are never kept: far less than their 4 GB.
    assert ws("fmxq_head_workspace", 8192, 128256, 1024, 1, True)[1] < 1 << 30
    assert ws("fmxq_head_workspace", 4, 0, 64, 1, True)[0] == "FMXQ_ERR_SHAPE"
    assert ws("fmxq_head_workspace", 4, 10, 64, 65, True)[0] == "FMXQ_ERR_SHAPE"
    assert ws("fmxq_quantized_matmul_grad_workspace", -1, 1, 1)[0] == "FMXQ_ERR_SHAPE"
    assert ws("fmxq_gather_qmm_grad_workspace", 1, -1, 1, 64)[0] == "FMXQ_ERR_SHAPE"
    assert ws("fmxq_moe_sort_workspace", 4, 2, 4096)[0] == "FMXQ_ERR_UNSUPPORTED"
    assert _lib.STATUS[_lib.load().fmxq_moe_sort_workspace(4, 2, 8, None)] == \
        "FMXQ_ERR_INVALID_ARGUMENT"


def test_torch_wrappers_refuse_cpu_tensors_and_shapes():
    bf = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.zeros(100, 8, dtype=torch.int32)
    s = torch.zeros(100, 1, dtype=torch.bfloat16)
    y = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: ops.head_cross_entropy(bf, w, s, s, y),
                 lambda: ops.head_distill(bf, w, s, s, y[:, None], bf[:, :1]),
                 lambda: ops.quantized_matmul_grad(bf, w, s, s),
                 lambda: ops.gather_qmm_grad(bf, w[None], s[None], s[None], y),
                 lambda: ops.moe_sort(bf, y[:, None], 4),
                 lambda: ops.moe_unsort(bf, y[:, None], bf[:, :1]),
                 lambda: ops.moe_unsort_grad(bf, bf, y[:, None], bf[:, :1]),
                 lambda: ops.moe_sort_grad(bf, y[:, None])):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError):
        ops.moe_sort(None, y, 4)


@pytest.mark.parametrize("M", [4, 5000])
@pytest.mark.parametrize("grad", [False, True])
def test_head_workspace_refuses_rows_of_no_width(M, grad):
    assert ws("fmxq_head_workspace", M, 100, 0, 1, grad)[0] == "FMXQ_ERR_SHAPE"
    assert ws("fmxq_head_workspace", 0, 100, 0, 1, grad) == ("FMXQ_OK", 0)


def test_a_gradient_needs_no_copy_of_a_large_weight():
    """The panel of dequantized weights is bounded, whatever their number."""
    for M, N, K in ((2048, 128256, 4096), (1025, 500000, 8192), (4096, 28672, 8192)):
        rc, n = ws("fmxq_quantized_matmul_grad_workspace", M, N, K)
        # A copy of dy, two parts of fp32 sums at most for that many tiles (three below 2048 rows
        # of 4096), and the panel.
        assert rc == "FMXQ_OK" and n <= 2 * M * (N + 8) + 3 * 4 * M * K + (513 << 20)


def test_gradients_reserve_no_copy_of_rows_that_are_read_as_they_are():
    rc, n = ws("fmxq_gather_qmm_grad_workspace", 65536, 64, 7168, 2048)
    assert rc == "FMXQ_OK" and n <= 4096
    rc, n = ws("fmxq_quantized_matmul_grad_workspace", 4096, 28672, 4096)
    assert rc == "FMXQ_OK" and n <= 28672 * 4096 * 2 + 4096
    # Rows of 7 values are copied to 8.
    assert ws("fmxq_gather_qmm_grad_workspace", 1000, 4, 7, 64)[1] >= 1000 * 8 * 2
    for name, sizes in (("fmxq_gather_qmm_grad_workspace", (0, 4, 7, 64)),
                        ("fmxq_quantized_matmul_grad_workspace", (0, 7, 64))):
        assert ws(name, *sizes) == ("FMXQ_OK", 0)


def test_moved_rows_need_their_bytes():
    """dy at an odd address: what the query reports does not do, and nothing is enqueued."""
    for M, N in ((4, 16), (40, 512)):
        n = ws("fmxq_quantized_matmul_grad_workspace", M, N, 64)[1]
        assert grad(dy=P + 2, M=M, N=N, n=n + M * N * 2 - 1) == "FMXQ_ERR_INVALID_ARGUMENT"
        n = ws("fmxq_gather_qmm_grad_workspace", M, 3, N, 64)[1]
        assert gather(dy=P + 2, S=M, N=N, n=n + M * N * 2 - 1) == "FMXQ_ERR_INVALID_ARGUMENT"


def test_sizes_that_no_launch_takes_are_refused_first():
    """More blocks than a launch has, with or without a workspace (its address is never used)."""
    M, K = (1 << 24) - 1, 1 << 21
    assert grad(M=M, K=K) == gather(S=M, K=K) == ce(M=M, K=K) == "FMXQ_ERR_SHAPE"
    assert gather(S=(1 << 24) - 1, E=1 << 22, K=4096) == "FMXQ_ERR_SHAPE"
    assert ws("fmxq_quantized_matmul_grad_workspace", M, 16, K)[0] == "FMXQ_ERR_SHAPE"
    assert ws("fmxq_gather_qmm_grad_workspace", M, 3, 16, K)[0] == "FMXQ_ERR_SHAPE"
    assert ws("fmxq_head_workspace", M, 100, K, 1, True)[0] == "FMXQ_ERR_SHAPE"
    # The loss alone has no such outputs.
    assert ws("fmxq_head_workspace", M, 100, K, 1, False)[0] == "FMXQ_OK"


def test_no_panel_where_its_offsets_do_not_fit():
    """K past what the panel's 32-bit offsets hold: tiles without a panel, which need no memory."""
    wide = 4180000
    rc, n = ws("fmxq_quantized_matmul_grad_workspace", 1025, 16, wide)
    assert rc == "FMXQ_OK" and n < 16 * wide * 2
    rc, n = ws("fmxq_head_workspace", 2000, 64, wide, 1, False)
    assert rc == "FMXQ_OK" and n < 64 * wide * 2


def test_the_sorts_histograms_do_not_grow_with_the_slots():
    """Every block reads all of them."""
    assert ws("fmxq_moe_sort_workspace", 1 << 23, 7, 2048) == ("FMXQ_OK", 512 * 2049 * 4)
    assert ws("fmxq_moe_sort_workspace", (1 << 24) - 1, 3, 8)[1] <= 512 * 9 * 4
    assert ws("fmxq_moe_sort_workspace", 0, 4, 8) == ("FMXQ_OK", 0)
