"""numpy restatement of the 4-bit KV cache (test infrastructure).

``encode`` / ``decode`` fix the numbers (64-bit arithmetic over the 16-bit
inputs), ``byte_of`` the bytes, one value at a time; ``append`` and ``rows``
apply them to a cache ``[N, L, Hkv, 2, R]`` of uint8.  Attention is the textbook
in float64 over the decoded rows.
"""
from __future__ import annotations

from typing import Tuple

import numpy as np

BLOCK = 16
GROUP = 32
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
LOW, TOP = -125, {"bf16": 125, "fp16": 13}


def record_bytes(dim: int) -> int:
    return 8 * dim + dim // 2


def encode(x: np.ndarray, dtype: str) -> Tuple[np.ndarray, np.ndarray]:
    """Rows ``[..., D]`` (float64) -> codes ``[..., D]`` and scale bytes
    ``[..., D/32]``."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(invalid="ignore"):
        a = np.abs(g).max(-1)
    finite = np.isfinite(g).all(-1)
    exps = np.arange(LOW, TOP[dtype] + 1)
    # the first exponent whose 7 * 2^e lies above the maximum, else the last
    at = np.searchsorted(np.ldexp(7.0, exps), np.where(finite, a, 0), side="right")
    e = exps[np.minimum(at, len(exps) - 1)]
    y = np.ldexp(np.abs(np.where(finite[..., None], g, 0)), -e[..., None])
    # the nearest grid value; of two equally near ones the even code
    away = np.abs(y[..., None] - GRID)
    even_first = np.where(away == away.min(-1, keepdims=True), np.arange(8) % 2, 2)
    code = even_first.argmin(-1).astype(np.uint8)
    code |= np.signbit(g).astype(np.uint8) << 3
    code = np.where(finite[..., None], code, 0).astype(np.uint8)
    scale = np.where(finite, e + 127, 255).astype(np.uint8)
    return code.reshape(x.shape), scale


def decode(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """Codes ``[..., D]`` and scale bytes -> float64."""
    v = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7]
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(int) - 127))
    return (v.reshape(*v.shape[:-1], -1, GROUP) * s[..., None]).reshape(v.shape)


def byte_of(side: int, dim: int, r: int, d: int) -> Tuple[int, int, int]:
    """(code byte, half of it, scale byte) in a record of dim ``d`` of token
    ``r``; side 0: K, 1: V."""
    if side == 0:
        per = 16 if dim == 64 else 32  # dims of a chunk
        at = (d // per * BLOCK + r) * (per // 2) + d % per // 2
    else:
        lane, o = divmod(d, dim // 16)
        w = min(8, dim // 16)
        at = (((o // w * 4 + r // 4) * 16 + lane) * 4 + r % 4) * (w // 2) + o % w // 2
    return at, d % 2, 8 * dim + d // GROUP * BLOCK + r


def _index(side: int, dim: int):
    """byte_of over a whole record: code bytes and halves ``[16, D]``, scale
    bytes ``[16, D/32]``."""
    t = [[byte_of(side, dim, r, d) for d in range(dim)] for r in range(BLOCK)]
    a = np.array(t)
    return a[..., 0], a[..., 1], a[:, ::GROUP, 2]


def append(key: np.ndarray, value: np.ndarray, cache: np.ndarray, slots: np.ndarray,
           dtype: str) -> None:
    """Rows ``[L, T, Hkv, D]`` (float64) into the cache, in place; slots
    outside the cache are skipped."""
    dim = key.shape[-1]
    for side, x in enumerate((key, value)):
        code_at, half, scale_at = _index(side, dim)
        codes, scales = encode(x, dtype)
        for t, s in enumerate(slots):
            if not 0 <= s < cache.shape[0] * BLOCK:
                continue
            b, r = divmod(int(s), BLOCK)
            rec = cache[b, :, :, side]  # [L, Hkv, R]
            c = codes[:, t]
            assert (half[r, 0::2] == 0).all() and (code_at[r, 0::2] == code_at[r, 1::2]).all()
            rec[..., code_at[r, 0::2]] = c[..., 0::2] | (c[..., 1::2] << 4)
            rec[..., scale_at[r]] = scales[:, t]


def rows(cache: np.ndarray, dim: int) -> Tuple[np.ndarray, np.ndarray]:
    """K and V of every slot of one layer ``[N, Hkv, 2, R]``, float64
    ``[N, 16, Hkv, D]``."""
    out = []
    for side in (0, 1):
        code_at, half, scale_at = _index(side, dim)
        rec = cache[:, :, side]
        codes = (rec[..., code_at] >> (4 * half)) & 15  # [N, Hkv, 16, D]
        out.append(decode(codes, rec[..., scale_at]).transpose(0, 2, 1, 3))
    return out[0], out[1]


def varlen_attention(q: np.ndarray, k_rows: np.ndarray, v_rows: np.ndarray, tables, cu_q, seq_lens,
                     scale: float, causal: bool) -> np.ndarray:
    """Queries ``[T, Hq, D]`` of sequence b at ``cu_q[b] .. cu_q[b + 1]``, the
    last of its ``seq_lens[b]`` tokens; a query without a key gives zeros."""
    T, hq, dim = q.shape
    hkv = k_rows.shape[2]
    out = np.zeros(q.shape)
    for b, n in enumerate(int(x) for x in seq_lens):
        t0, t1 = int(cu_q[b]), int(cu_q[b + 1])
        m = t1 - t0
        if m == 0 or n == 0:
            continue
        ids = np.asarray(tables[b][:-(-n // BLOCK)])
        # (heads first and dense: numpy multiplies strided matrices without its BLAS)
        k, v = (np.ascontiguousarray(x[ids].reshape(-1, hkv, dim)[:n].swapaxes(0, 1))
                for x in (k_rows, v_rows))
        seen = np.ones((m, n), bool)
        if causal:
            seen = np.arange(n)[None, :] <= (n - m + np.arange(m))[:, None]
        for h in range(hq):
            s = np.ascontiguousarray(q[t0:t1, h]) @ k[h * hkv // hq].T * scale
            s[~seen] = -np.inf
            top = s.max(-1, keepdims=True)
            p = np.exp(s - np.where(np.isfinite(top), top, 0))
            l = p.sum(-1, keepdims=True)
            out[t0:t1, h] = np.where(l > 0, p @ v[h * hkv // hq] / np.where(l > 0, l, 1), 0)
    return out
