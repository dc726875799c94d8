"""What log probabilities through a quantized head refuse, before anything is enqueued (CPU)."""
import ctypes

import pytest

from fastmlx_amd import _lib

P = 4096  # an aligned address that is never read


def status(name, *args):
    return _lib.STATUS[getattr(_lib.load(), name)(*args)]


def scores(h=P, w=P, s=P, ids=P, logp=P, ent=P, lse=P, ti=P, tl=P, M=4, V=100, K=64, k=2, top=3, T=1.0, group=64,
           bits=4, work=P, n=1 << 40):
    return status("fmxq_head_logprobs", h, w, s, P, ids, logp, ent, lse, ti, tl, M, V, K, k, top, T, group, bits,
                  work, n, None)


def grads(h=P, w=P, s=P, ids=P, logp=P, ent=P, lse=P, gl=P, ge=P, dh=P, M=4, V=100, K=64, k=2, T=1.0, group=64,
          bits=4, work=P, n=1 << 40):
    return status("fmxq_head_logprobs_grad", h, w, s, P, ids, logp, ent, lse, gl, ge, dh, M, V, K, k, T, group,
                  bits, work, n, None)


BOTH = [
    (dict(bits=3), "UNSUPPORTED"), (dict(group=16), "UNSUPPORTED"), (dict(K=65), "SHAPE"), (dict(K=0), "SHAPE"),
    (dict(M=-1), "SHAPE"), (dict(V=-1), "SHAPE"), (dict(V=0), "SHAPE"), (dict(M=1 << 25), "SHAPE"),
    (dict(k=65), "SHAPE"), (dict(k=-1), "SHAPE"), (dict(V=1 << 31), "SHAPE"),
    (dict(T=0.0), "INVALID_ARGUMENT"), (dict(T=-1.0), "INVALID_ARGUMENT"), (dict(T=float("nan")), "INVALID_ARGUMENT"),
    (dict(T=float("inf")), "INVALID_ARGUMENT"), (dict(h=None), "INVALID_ARGUMENT"), (dict(w=None), "INVALID_ARGUMENT"),
    (dict(ids=None), "INVALID_ARGUMENT"), (dict(logp=None), "INVALID_ARGUMENT"), (dict(ent=None), "INVALID_ARGUMENT"),
    (dict(lse=None), "INVALID_ARGUMENT"), (dict(h=P + 2), "INVALID_ARGUMENT"), (dict(w=P + 4), "INVALID_ARGUMENT"),
    (dict(ids=P + 2), "INVALID_ARGUMENT"), (dict(logp=P + 2), "INVALID_ARGUMENT"), (dict(s=P + 1), "INVALID_ARGUMENT"),
    (dict(work=None), "INVALID_ARGUMENT"), (dict(work=P + 8), "INVALID_ARGUMENT"), (dict(n=100), "INVALID_ARGUMENT"),
]


@pytest.mark.parametrize("kw,want", BOTH + [
    (dict(top=-1), "SHAPE"), (dict(top=65), "SHAPE"), (dict(V=2), "SHAPE"), (dict(ti=None), "INVALID_ARGUMENT"),
    (dict(tl=None), "INVALID_ARGUMENT"), (dict(ti=P + 2), "INVALID_ARGUMENT")])
def test_scores_refuse(kw, want):
    assert scores(**kw) == "FMXQ_ERR_" + want


@pytest.mark.parametrize("kw,want", BOTH + [
    (dict(k=0), "SHAPE"), (dict(gl=None), "INVALID_ARGUMENT"), (dict(dh=None), "INVALID_ARGUMENT"),
    (dict(dh=P + 8), "INVALID_ARGUMENT"), (dict(ge=P + 2), "INVALID_ARGUMENT")])
def test_grads_refuse(kw, want):
    assert grads(**kw) == "FMXQ_ERR_" + want


def ws(name, *sizes):
    n = ctypes.c_size_t()
    rc = getattr(_lib.load(), name)(*sizes, ctypes.byref(n))
    return _lib.STATUS[rc], n.value


def test_workspaces():
    assert ws("fmxq_head_logprobs_workspace", 0, 0, 0, 0, 0) == ("FMXQ_OK", 0)
    assert ws("fmxq_head_logprobs_grad_workspace", 0, 0, 0, 1) == ("FMXQ_OK", 0)
    plain, top = (ws("fmxq_head_logprobs_workspace", 2048, 128256, 4096, 1, t)[1] for t in (0, 20))
    assert 0 < plain < top < (3 << 30)
    # Rows go in chunks: more of them take no more memory.
    assert ws("fmxq_head_logprobs_workspace", 1 << 20, 128256, 4096, 1, 20)[1] < (4 << 30)
    assert ws("fmxq_head_logprobs_workspace", 4, 100, 64, 2, 101)[0] == "FMXQ_ERR_SHAPE"
    for name, sizes in (("fmxq_head_logprobs_workspace", (4, 100, 64, 2, 3)),
                        ("fmxq_head_logprobs_grad_workspace", (4, 100, 64, 2))):
        assert _lib.STATUS[getattr(_lib.load(), name)(*sizes, None)] == "FMXQ_ERR_INVALID_ARGUMENT"
