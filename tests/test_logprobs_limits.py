"""The product that log probabilities of few rows take fits a launch at every vocabulary (CPU)."""
import ctypes

import pytest

from fastmlx_amd import _lib


@pytest.mark.parametrize("V,tile", [(2 ** 27 - 256, 16), (2 ** 27, 32), (2 ** 27 + 5000, 32), (2 ** 31 - 1, 32)])
@pytest.mark.parametrize("M", [1, 4])
def test_tiles_of_large_vocabularies(M, V, tile):
    """Blocks of 16 tokens while they are fewer than 2^23, of 32 above: 16 bytes of workspace a tile."""
    n = ctypes.c_size_t()
    assert _lib.load().fmxq_head_logprobs_workspace(M, V, 32, 1, 0, ctypes.byref(n)) == 0
    tiles = (V + 255) // 256 * 256 // tile
    assert M * tiles * 16 <= n.value < M * tiles * 16 + 2 ** 20
