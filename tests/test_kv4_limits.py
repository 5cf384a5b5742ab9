"""The 4-bit cache's entry points at the edges of their arguments, without a
GPU: every call here is refused on the host."""
import numpy as np
import pytest

from aegaeon_amd import _lib

INVALID = -1


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.fixture(scope="module")
def ptr():
    raw = np.zeros(1 << 16, dtype=np.uint8)
    yield (raw.ctypes.data + 15) // 16 * 16
    del raw


BAD_SCALES = [float("nan"), float("inf"), float("-inf"), 3e38, -3e38]


@pytest.mark.parametrize("scale", BAD_SCALES)
def test_decode_refuses_a_scale_that_overflows(lib, ptr, scale):
    """Not finite, or not times log2 e: a score of zero or a masked one would give
    NaN."""
    p = ptr
    assert lib.aegkv_kv4_decode_attention(p, 1024, p, 1024, p, 17 * 4 * 128, 8, p, 4, p, 2, 64, 8,
                                          4, 128, scale, 0, 8, p, 1 << 30, None) == INVALID
    assert lib.aegkv_kv4_decode_attention_planned(p, 1024, p, 1024, p, 17 * 4 * 128, 8, p, 1 << 16,
                                                  p, 2, 64, 8, 4, 128, scale, 0, 8, p, 1 << 30,
                                                  None) == INVALID
