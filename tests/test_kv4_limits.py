"""The 4-bit cache's entry points at the edges of their arguments, without a
GPU: every call here is refused on the host."""
import numpy as np
import pytest

from aegaeon_amd import _lib

INVALID, UNSUPPORTED = -1, -6


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


def test_several_queries_refuse_lengths_whose_last_step_passes_32_bits(lib):
    """A step of two key tiles ends up to 127 keys past the last one, the loads ahead
    two tiles further."""
    size = lib.aegkv_kv4_varlen_attention_workspace_size
    for longest in (2 ** 31 - 1, 2 ** 31 - 65, 2 ** 31 - 128, 2 ** 31 - 256):
        for new in (1, 20, 600):
            assert size(1, new, new, longest, 8, 2, 128, 0) == UNSUPPORTED


def test_several_queries_refuse_head_counts_past_65535(lib):
    """As the decode attention does: the row tiles of larger ones would pass 64 bits."""
    size = lib.aegkv_kv4_varlen_attention_workspace_size
    assert size(1, 1, 1, 64, 65536, 1, 128, 0) == UNSUPPORTED
    assert size(1, 1, 1, 64, 1 << 20, 1 << 20, 128, 0) == UNSUPPORTED
    assert size(2 ** 31 - 1, 2 ** 63 - 1, 1, 64, 2 ** 31 - 1, 2 ** 31 - 1, 128, 0) == UNSUPPORTED
