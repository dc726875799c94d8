"""Sizes whose launches together are more blocks than one takes are refused before anything is enqueued (CPU)."""
import ctypes

import pytest

from fastmlx_amd import _lib


def lora_grad_workspace(M, N, K, E, r):
    n = ctypes.c_size_t()
    return _lib.STATUS[_lib.load().fmxq_quantized_matmul_lora_grad_workspace(M, N, K, E, r, ctypes.byref(n))]


# The turned copies of A and B share a launch of at most 2^23 blocks of 32 by 32 values: (K / 32 + N / 32) (r / 32) E.
@pytest.mark.parametrize("N,K,E,r,want", [
    (16384, 16384, 2048, 128, "SHAPE"), (16384, 16352, 2048, 128, "OK"), (32704, 32, 2048, 128, "OK"),
    (30000, 20480, 2048, 96, "SHAPE"), (21824, 21824, 2048, 96, "OK"),
    # The outer products: (ceil(K / 128) + ceil(N / 128)) E of one part each.
    (262144, 262144, 2048, 8, "SHAPE")])
def test_adapters_of_both_sides_together(N, K, E, r, want):
    got = lora_grad_workspace(1, N, K, E, r)
    assert got == ("FMXQ_OK" if want == "OK" else "FMXQ_ERR_" + want)


def test_one_padded_copy_of_dy():
    """Rows that are no multiple of 8 values are copied once: into the input gradient's own place."""
    def bytes_of(name, *sizes):
        n = ctypes.c_size_t()
        assert getattr(_lib.load(), name)(*sizes, ctypes.byref(n)) == 0
        return n.value

    # The adapters' own parts are the same for 4097 and for 4104 values, but for the outer products' parts of 7 rows.
    M, K = 600, 512
    odd, even = (bytes_of("fmxq_quantized_matmul_lora_grad_workspace", M, N, K, 1, 8) -
                 bytes_of("fmxq_quantized_matmul_grad_workspace", M, N, K) for N in (4097, 4104))
    assert odd <= even
