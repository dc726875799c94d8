"""What adapters beside quantized products and gradient clipping refuse, before anything is
enqueued (CPU)."""
import ctypes

import pytest

from fastmlx_amd import _lib

P = 4096  # an aligned address that is never read


def status(name, *args):
    return _lib.STATUS[getattr(_lib.load(), name)(*args)]


def lora(x=P, w=P, a=P, b=P, ids=P, ls=P, y=P, M=4, N=16, K=64, E=3, r=8, group=64, bits=4, work=P,
         n=1 << 40):
    return status("fmxq_quantized_matmul_lora", x, w, P, P, a, b, ids, ls, y, M, N, K, E, r, group, bits,
                  work, n, None)


def lora_grad(dy=P, x=P, w=P, a=P, b=P, ids=P, ls=P, dx=P, da=P, db=P, M=4, N=16, K=64, E=3, r=8, group=64,
              bits=4, work=P, n=1 << 40):
    return status("fmxq_quantized_matmul_lora_grad", dy, x, w, P, P, a, b, ids, ls, dx, da, db, M, N, K, E,
                  r, group, bits, work, n, None)


BOTH = [
    (dict(bits=3), "UNSUPPORTED"), (dict(group=16), "UNSUPPORTED"), (dict(K=65), "SHAPE"),
    (dict(K=0), "SHAPE"), (dict(M=-1), "SHAPE"), (dict(N=-1), "SHAPE"), (dict(E=0), "UNSUPPORTED"),
    (dict(E=2049), "UNSUPPORTED"), (dict(E=-1), "UNSUPPORTED"), (dict(r=0), "UNSUPPORTED"),
    (dict(r=12), "UNSUPPORTED"), (dict(r=136), "UNSUPPORTED"), (dict(r=-8), "UNSUPPORTED"),
    (dict(M=1 << 25), "SHAPE"), (dict(N=1 << 22), "SHAPE"), (dict(M=(1 << 24) - 1, N=1 << 21), "SHAPE"),
    (dict(x=None), "INVALID_ARGUMENT"), (dict(w=None), "INVALID_ARGUMENT"), (dict(a=None), "INVALID_ARGUMENT"),
    (dict(b=None), "INVALID_ARGUMENT"), (dict(ids=None), "INVALID_ARGUMENT"), (dict(ls=None), "INVALID_ARGUMENT"),
    (dict(x=P + 2), "INVALID_ARGUMENT"), (dict(w=P + 4), "INVALID_ARGUMENT"), (dict(a=P + 8), "INVALID_ARGUMENT"),
    (dict(b=P + 8), "INVALID_ARGUMENT"), (dict(ids=P + 2), "INVALID_ARGUMENT"), (dict(ls=P + 2), "INVALID_ARGUMENT"),
    (dict(work=None), "INVALID_ARGUMENT"), (dict(work=P + 8), "INVALID_ARGUMENT"), (dict(n=100), "INVALID_ARGUMENT"),
]


@pytest.mark.parametrize("kw,want", BOTH + [(dict(y=None), "INVALID_ARGUMENT"), (dict(y=P + 8), "INVALID_ARGUMENT")])
def test_lora_refuses(kw, want):
    assert lora(**kw) == "FMXQ_ERR_" + want


@pytest.mark.parametrize("kw,want", BOTH + [
    (dict(dy=None), "INVALID_ARGUMENT"), (dict(dy=P + 1), "INVALID_ARGUMENT"), (dict(dx=None), "INVALID_ARGUMENT"),
    (dict(dx=P + 8), "INVALID_ARGUMENT"), (dict(da=None), "INVALID_ARGUMENT"), (dict(da=P + 4), "INVALID_ARGUMENT"),
    (dict(db=None), "INVALID_ARGUMENT"), (dict(db=P + 8), "INVALID_ARGUMENT"),
    (dict(E=2048, r=128, N=1 << 21), "SHAPE")])
def test_lora_grad_refuses(kw, want):
    assert lora_grad(**kw) == "FMXQ_ERR_" + want


def ws(name, *sizes):
    n = ctypes.c_size_t()
    rc = getattr(_lib.load(), name)(*sizes, ctypes.byref(n))
    return _lib.STATUS[rc], n.value


@pytest.mark.parametrize("name", ["fmxq_quantized_matmul_lora_workspace", "fmxq_quantized_matmul_lora_grad_workspace"])
def test_lora_workspaces(name):
    assert ws(name, 0, 16, 64, 3, 8) == ("FMXQ_OK", 0)
    assert ws(name, 0, 0, 0, 1, 8) == ("FMXQ_OK", 0)
    rc, n = ws(name, 300, 16, 64, 3, 8)
    assert rc == "FMXQ_OK" and n >= 300 * 8 * 4
    assert ws(name, -1, 16, 64, 3, 8)[0] == "FMXQ_ERR_SHAPE"
    assert ws(name, 4, 16, 64, 3, 7)[0] == "FMXQ_ERR_UNSUPPORTED"
    assert _lib.STATUS[getattr(_lib.load(), name)(4, 16, 64, 3, 8, None)] == "FMXQ_ERR_INVALID_ARGUMENT"


def clip(n=2, grads=(P, 2 * P), outs=(3 * P, 4 * P), counts=(8, 8), bf16=(0, 1), most=1.0, norm=P, work=P,
         size=1 << 20):
    def arr(t, v):
        return None if v is None else (t * len(v))(*v)
    g, o = arr(ctypes.c_void_p, grads), arr(ctypes.c_void_p, outs)
    return status("fmxq_clip_grad_norm", g, o, arr(ctypes.c_int64, counts), arr(ctypes.c_int, bf16), n, most,
                  norm, work, size, None)


@pytest.mark.parametrize("kw,want", [
    (dict(n=-1), "SHAPE"), (dict(n=(1 << 20) + 1), "SHAPE"), (dict(grads=None), "INVALID_ARGUMENT"),
    (dict(outs=None), "INVALID_ARGUMENT"), (dict(counts=None), "INVALID_ARGUMENT"),
    (dict(bf16=None), "INVALID_ARGUMENT"), (dict(norm=None), "INVALID_ARGUMENT"),
    (dict(norm=P + 2), "INVALID_ARGUMENT"), (dict(work=None), "INVALID_ARGUMENT"),
    (dict(work=P + 8), "INVALID_ARGUMENT"), (dict(size=100), "INVALID_ARGUMENT"),
    (dict(counts=(8, -1)), "SHAPE"), (dict(counts=(8, 1 << 41)), "SHAPE"), (dict(grads=(P, None)), "INVALID_ARGUMENT"),
    (dict(grads=(P + 2, 2 * P)), "INVALID_ARGUMENT"), (dict(grads=(P, 2 * P + 1)), "INVALID_ARGUMENT"),
    (dict(outs=(3 * P + 2, 4 * P)), "INVALID_ARGUMENT"), (dict(outs=(3 * P, None)), "INVALID_ARGUMENT"),
    (dict(most=-1.0), "INVALID_ARGUMENT"), (dict(most=float("nan")), "INVALID_ARGUMENT"),
    # Results over each other, a gradient over another's result, and over its own but for a shift.
    (dict(outs=(3 * P, 3 * P)), "INVALID_ARGUMENT"), (dict(outs=(3 * P, 3 * P + 16)), "INVALID_ARGUMENT"),
    (dict(outs=(2 * P, P)), "INVALID_ARGUMENT"), (dict(outs=(P + 4, 4 * P)), "INVALID_ARGUMENT"),
    (dict(grads=(P, P), outs=(P, P)), "INVALID_ARGUMENT"),
    (dict(grads=(P, P + 16), outs=(P, 4 * P)), "INVALID_ARGUMENT")])
def test_clip_refuses(kw, want):
    assert clip(**kw) == "FMXQ_ERR_" + want


def test_clip_workspace():
    assert ws("fmxq_grad_norm_workspace")[0] == "FMXQ_OK"
    assert status("fmxq_grad_norm_workspace", None) == "FMXQ_ERR_INVALID_ARGUMENT"
