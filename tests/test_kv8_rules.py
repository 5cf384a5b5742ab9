"""The 8-bit cache's rules without a GPU: which tokens join a block at once, how far
a held value may be off, and what the outputs of a rotating append may not share."""
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


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rises", [0, 1, 2, 5])
def test_how_far_a_held_value_is_off(dtype, rises):
    """Rounded once: 2^-4 of itself or 2^-10 of the scale.  After rises of the block's
    exponent: 2^-4 of itself or less than 2^-9 of the scale, as roundings at scales
    that double add up to less than twice the last one's.  (Exact in 64 bits.)"""
    rng = np.random.default_rng(rises)
    D, past = 64, 0
    for trial in range(60):
        cache = np.zeros((1, 1, k8.block_bytes(1, D)), dtype=np.uint8)
        x = np.exp(rng.uniform(-10, 0, size=(1, 1, 1, D))) * rng.choice([-1, 1], size=(1, 1, 1, D))
        x[..., 0] = 1.0
        x *= 2.0 ** -6
        k8.append(x, x, cache, np.array([0]), dtype)
        for i in range(rises):
            y = np.full((1, 1, 1, D), 2.0 ** -6 * 2.0 ** (i + 1))
            k8.append(y, y, cache, np.array([1 + i]), dtype)
        e = int(cache[0, 0, 32 * D]) - 127
        assert e == -14 + rises
        held = k8.rows(cache[:, 0], 1, D)[0][0, 0, 0]
        off, own = np.abs(held - x[0, 0, 0]), 2.0 ** -4 * np.abs(x[0, 0, 0])
        past += int((off > np.maximum(own, 2.0 ** (e - 10))).sum())
        assert (np.maximum(off - own, 0) == 0)[off >= 2.0 ** (e - 9)].all()
    assert (past > 0) == (rises > 0)  # the bound of one rounding does not hold for several


def test_values_past_the_largest_are_held_as_that():
    cache = np.zeros((1, 1, k8.block_bytes(1, 64)), dtype=np.uint8)
    x = np.full((1, 1, 1, 64), 65504.0)
    k8.append(x, -x, cache, np.array([0]), "fp16")
    k, v = k8.rows(cache[:, 0], 1, 64)
    assert (k[0, 0] == 57344.0).all() and (v[0, 0] == -57344.0).all()


def test_a_token_written_over_leaves_the_blocks_exponent():
    cache = np.zeros((1, 1, k8.block_bytes(1, 64)), dtype=np.uint8)
    for place, size in ((0, 1.0), (1, 1000.0), (1, 1.0)):
        x = np.full((1, 1, 1, 64), size)
        k8.append(x, x, cache, np.array([place]), "bf16")
    assert int(cache[0, 0, 32 * 64]) - 127 == 2   # 1000 <= 448 * 2^2, where 1.0 alone has -8


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
