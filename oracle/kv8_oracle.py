"""numpy restatement of the 8-bit KV cache and of the position rotation (test
infrastructure).

``encode`` / ``decode`` fix the numbers (64-bit arithmetic over a list of the
codes' values), ``byte_of`` the bytes, one value at a time; ``append`` and
``rows`` apply them to a cache ``[N, L, R]`` of uint8.  ``turned`` is the rotation
in float32, every operation rounded by itself.  Attention is kv4_oracle's
textbook in float64 over the decoded rows.
"""
from __future__ import annotations

from functools import lru_cache
from itertools import groupby
from typing import Tuple

import numpy as np

BLOCK = 16
LARGEST = 448.0
LOW, TOP = {"bf16": -117, "fp16": -15}, {"bf16": 119, "fp16": 7}
NAN = 0xFF
# the values of codes 0 .. 126: four exponent bits (bias 7), three mantissa bits
GRID = np.array([m * 2.0 ** -9 if p == 0 else (8 + m) * 2.0 ** (p - 10)
                 for p in range(16) for m in range(8)][:127])


def block_bytes(heads: int, dim: int) -> int:
    return 32 * heads * dim + -(-4 * heads // 128) * 128


def exponent(x: np.ndarray, dtype: str) -> int:
    """Of the finite values among x."""
    a = np.abs(x[np.isfinite(x)]).max(initial=0.0)
    e = LOW[dtype]
    while e < TOP[dtype] and a > LARGEST * 2.0 ** e:
        e += 1
    return e


def encode(x: np.ndarray, e: int) -> np.ndarray:
    """Values to code bytes under exponent e."""
    fine = np.isfinite(x)
    y = np.abs(np.ldexp(np.where(fine, x, 0).astype(np.float64), -e))
    hi = np.clip(np.searchsorted(GRID, y), 1, 126)  # GRID[hi - 1] <= y <= GRID[hi], if in range
    below, above = y - GRID[hi - 1], GRID[hi] - y
    code = np.where((below < above) | ((below == above) & (hi % 2 == 1)), hi - 1, hi)
    code = np.where(np.signbit(x), code | 0x80, code)
    return np.where(fine, code, NAN).astype(np.uint8)


def decode(codes: np.ndarray, e) -> np.ndarray:
    v = np.append(GRID, np.nan)[codes & 0x7F]
    return np.ldexp(np.where(codes & 0x80, -v, v), e)


def byte_of(side: int, dim: int, r: int, d: int) -> int:
    """Byte of dim ``d`` of token ``r`` in a side's codes (0: K, 1: V)."""
    if side == 0:
        return d // 16 * 256 + r * 16 + d % 16
    lane, o = divmod(d, dim // 16)
    return ((o // 4 * 4 + r // 4) * 16 + lane) * 16 + o % 4 * 4 + r % 4


@lru_cache(maxsize=None)
def _index(side: int, dim: int) -> np.ndarray:
    return np.array([[byte_of(side, dim, r, d) for d in range(dim)] for r in range(BLOCK)])


def append(key: np.ndarray, value: np.ndarray, cache: np.ndarray, slots: np.ndarray,
           dtype: str) -> None:
    """Rows ``[L, T, Hkv, D]`` (float32 or float64) into the cache, in place;
    slots outside the cache are skipped, and tokens of a block join it at once
    where no other block's lie between them."""
    L, T, H, D = key.shape
    slots = [int(s) for s in slots]
    written = [t for t in range(T) if 0 <= slots[t] < cache.shape[0] * BLOCK]
    for blk, run in groupby(written, key=lambda t: slots[t] // BLOCK):
        place = {slots[t] % BLOCK: t for t in run}  # the later of two
        for layer in range(L):
            for h in range(H):
                for side, x in enumerate((key, value)):
                    _put(cache[blk, layer], side, H, D, h,
                         {r: x[layer, t, h] for r, t in place.items()}, dtype)


def _put(layer_block, side, H, D, h, new, dtype):
    at = (2 * h + side) * 16 * D + _index(side, D)  # [16, D]
    s = 32 * H * D + 4 * h
    e = exponent(np.stack(list(new.values())), dtype)
    anew = 0 in new
    # (one that no append wrote counts as the nearer bound)
    held = min(max(int(layer_block[s + side]) - 127, LOW[dtype]), TOP[dtype])
    codes = np.zeros((BLOCK, D), np.uint8)
    if not anew:
        codes = layer_block[at]
        if held >= e:
            e = held
        else:
            codes = encode(decode(codes, held), e)
    codes[list(new)] = encode(np.stack(list(new.values())), e)
    layer_block[at] = codes
    layer_block[s + side] = e + 127
    if side == 1:
        nan = any(not np.isfinite(x).all() for x in new.values())
        if anew or nan:
            layer_block[s + 2] = nan


def rows(cache: np.ndarray, heads: int, dim: int) -> Tuple[np.ndarray, np.ndarray]:
    """K and V of every slot of one layer ``[N, R]``, float64 ``[N, 16, Hkv, D]``."""
    out = []
    for side in (0, 1):
        at = _index(side, dim)
        per_head = []
        for h in range(heads):
            e = cache[:, 32 * heads * dim + 4 * h + side].astype(int) - 127
            per_head.append(decode(cache[:, (2 * h + side) * 16 * dim + at], e[:, None, None]))
        out.append(np.stack(per_head, 2))
    return out[0], out[1]


def turned(x: np.ndarray, positions: np.ndarray, table: np.ndarray,
           interleaved: bool) -> np.ndarray:
    """Rows ``[T, H, D]`` (16-bit values) turned by their positions, float32; a
    position outside the table gives NaN."""
    x = x.astype(np.float32)
    half = table.shape[1] // 2
    inside = (positions >= 0) & (positions < len(table))
    t = np.where(inside[:, None], table[np.where(inside, positions, 0)], np.float32(np.nan))
    cos, sin = t[:, None, :half], t[:, None, half:]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
    else:
        a, b = x[..., :half], x[..., half:2 * half]
    u, w = a * cos - b * sin, b * cos + a * sin
    out = x.copy()
    if interleaved:
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = u, w
    else:
        out[..., :half], out[..., half:2 * half] = u, w
    return out
