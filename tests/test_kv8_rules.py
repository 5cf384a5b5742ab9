"""The 8-bit cache's rules without a GPU: which tokens join a block at once, and what
the outputs of a rotating append may not share."""
import numpy as np
import pytest

from aegaeon_amd import rotary
from oracle import kv8_oracle as k8


@pytest.mark.parametrize("skipped", [[-1], [64], [-9, 1000, -1]])
def test_skipped_rows_do_not_part_a_blocks_tokens(skipped):
    """The same bytes as without them: one exponent at once, no value rounded twice."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((1, 3, 2, 64)) * np.array([1.0, 2.0 ** -9, 500.0])[:, None, None]
    want = np.zeros((4, 1, k8.block_bytes(2, 64)), dtype=np.uint8)
    k8.append(x, -x, want, np.array([16, 17, 18]), "bf16")
    n = len(skipped)
    slots = np.array([16, *skipped, 17, *skipped, 18])
    rows = np.full((1, len(slots), 2, 64), 7e4)
    rows[:, [0, n + 1, 2 * n + 2]] = x
    got = np.zeros_like(want)
    k8.append(rows, -rows, got, slots, "bf16")
    assert np.array_equal(got, want)


def test_outputs_of_a_rotation_lie_clear_of_what_the_call_uses():
    """The addresses that a call's outputs may not share; neighbours that touch are
    clear."""
    first, n = 1 << 40, 1 << 20
    others = [("table", 1 << 60, (1 << 60) + 64), ("key_cache", first, first + n)]
    rotary._check_clear([("out", first - 64, first), ("out_key", first + n, first + n + 64)], others)
    for a, b in ((first - 64, first + 2), (first + n - 2, first + n + 64), (first - 2, first + n + 2),
                 (first + 64, first + 128)):
        with pytest.raises(ValueError, match="out_key overlaps key_cache"):
            rotary._check_clear([("out_key", a, b)], others)
    with pytest.raises(ValueError, match="out overlaps table"):
        rotary._check_clear([("out", 1 << 60, (1 << 60) + 2)], others)
