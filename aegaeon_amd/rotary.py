"""Queries and keys turned by their positions on the way into the cache, in one
launch per layer where vLLM's rotary embedding and
:func:`attention.reshape_and_cache_flash` are two and more (reached from
aegaeon/aegaeon/worker.py:517-523):

* :func:`rotary_table` — the angles' cosines and sines, once per model;
* :func:`rotary_and_cache` — the turned queries, and the turned keys and the
  values in the 16-bit cache (:func:`kv8.rotary_and_cache_kv8`: the 8-bit one).

Everything is enqueued on the current torch stream.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._gpu import device_guard, raw_stream
from .attention import _DTYPES, _check_cache_view, _check_on, _check_rows


def rotary_table(max_positions: int, rotary_dim: int, base: float = 10000.0,
                 device="cuda") -> torch.Tensor:
    """``[max_positions, rotary_dim]`` float32: the cosines of a position's
    angles ``position * base^(-2 i / rotary_dim)``, i below ``rotary_dim / 2``,
    then their sines; the angles in 64 bits."""
    if rotary_dim <= 0 or rotary_dim % 16:
        raise ValueError("rotary_dim must be a positive multiple of 16")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    angle = torch.arange(max_positions, dtype=torch.float64)[:, None] \
        * float(base) ** (-i / rotary_dim)
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


def _dense_rows(x: torch.Tensor, name: str, dev: torch.device, strides, head_dim: int) -> None:
    if x.get_device() != dev.index or strides[2] != 1 or strides[1] != head_dim:
        _check_on(x, name, dev)
        _check_rows(x, name)


def _check_apart(name: str, written, read, same: Tuple[str, ...]) -> None:
    """``written``, rows given as (first byte, token stride, row bytes, byte past
    the last), may be those of ``read`` that ``same`` names, and shares no byte with
    the others."""
    a, step, row, b = written
    for of, (c, other_step, other_row, d) in read:
        if a >= d or c >= b or (a == c and step == other_step and of in same):
            continue
        # slices of one wider buffer (a fused projection's columns) lie side by side
        if step == other_step and step > 0:
            off = (c - a) % step
            if off >= row and off + other_row <= step:
                continue
        raise ValueError(f"{name} overlaps {of}")


def _check_clear(written, others) -> None:
    """No row of ``written`` lies in a tensor of ``others``, whatever gaps its blocks
    have; both (name, first byte, byte past the last)."""
    for name, a, b in written:
        for of, c, d in others:
            if a < d and c < b:
                raise ValueError(f"{name} overlaps {of}")


def _turn_args(query, key, value, slot_mapping, positions, table, interleaved, out, out_key, dev,
               key_in_place: bool, caches):
    """The checks that both caches' calls share (``caches``: as :func:`_check_clear`'s
    others): the leading arguments of the C entries (kept to one look-up each: a decode
    step's call is bound by its host time), the turned queries' tensor and what must
    outlive the call."""
    qs, ks, dtype = query.shape, key.shape, query.dtype
    if len(qs) != 3 or len(ks) != 3 or value.shape != ks or ks[0] != qs[0] or ks[2] != qs[2]:
        raise ValueError("query must be [T, Hq, D], key and value [T, Hkv, D] with its tokens "
                         "and head_dim")
    if dtype not in _DTYPES or key.dtype != dtype or value.dtype != dtype:
        raise ValueError("query, key and value must share a bf16/fp16 dtype")
    T, Hq, D = qs
    Hkv = ks[1]
    qt, kt, vt = query.stride(), key.stride(), value.stride()
    _dense_rows(query, "query", dev, qt, D)
    _dense_rows(key, "key", dev, kt, D)
    _dense_rows(value, "value", dev, vt, D)
    for x, n in ((slot_mapping, "slot_mapping"), (positions, "positions")):
        if x.get_device() != dev.index:
            _check_on(x, n, dev)
        if x.dtype != torch.int64 or x.dim() != 1 or x.numel() < T:
            raise ValueError(f"{n} must be an int64 GPU tensor with an entry for each of the {T} "
                             "tokens")
    if table.get_device() != dev.index:
        _check_on(table, "table", dev)
    ts = table.shape
    if table.dtype != torch.float32 or len(ts) != 2 or not table.is_contiguous() or ts[0] == 0 \
            or not 0 < ts[1] <= D:
        raise ValueError("table must be a contiguous float32 tensor [positions, rotary_dim] with "
                         f"rows of up to head_dim {D} entries")
    qp, kp, vp = query.data_ptr(), key.data_ptr(), value.data_ptr()
    q_row, k_row = 2 * Hq * D, 2 * Hkv * D
    given, read, rows = out is not None, (), ()
    if (given or out_key is not None) and T > 0:
        read = [("query", (qp, 2 * qt[0], q_row, qp + 2 * (T - 1) * qt[0] + q_row)),
                ("key", (kp, 2 * kt[0], k_row, kp + 2 * (T - 1) * kt[0] + k_row)),
                ("value", (vp, 2 * vt[0], k_row, vp + 2 * (T - 1) * vt[0] + k_row))]
    if given:
        ot = out.stride()
        if out.shape != qs or out.dtype != dtype:
            raise ValueError(f"out must have query's shape and dtype {tuple(qs)}, {dtype}")
        _dense_rows(out, "out", dev, ot, D)
        op, ot = out.data_ptr(), ot[0]
        if T > 0:
            if T > 1 and 2 * ot < q_row:
                raise ValueError("out's rows overlap each other")
            written = (op, 2 * ot, q_row, op + 2 * (T - 1) * ot + q_row)
            _check_apart("out", written, read, ("query",))
            read.append(("out", written))
            rows = (("out", op, written[3]),)
    else:
        out = query.new_empty(qs)
        op, ot = out.data_ptr(), Hq * D
    okp, okt = None, 0
    if out_key is not None:
        okt = out_key.stride()
        if out_key.shape != ks or out_key.dtype != dtype:
            raise ValueError(f"out_key must have key's shape and dtype {tuple(ks)}, {dtype}")
        _dense_rows(out_key, "out_key", dev, okt, D)
        okp, okt = out_key.data_ptr(), okt[0]
        if T > 1 and 2 * okt < k_row:
            raise ValueError("out_key's rows overlap each other")
        if T > 0:
            end = okp + 2 * (T - 1) * okt + k_row
            _check_apart("out_key", (okp, 2 * okt, k_row, end), read,
                         ("key",) if key_in_place else ())
            rows += (("out_key", okp, end),)
    slots, positions = slot_mapping.contiguous(), positions.contiguous()
    sp, pp, tp = slots.data_ptr(), positions.data_ptr(), table.data_ptr()
    if rows:
        _check_clear(rows, (("slot_mapping", sp, sp + 8 * T), ("positions", pp, pp + 8 * T),
                            ("table", tp, tp + 4 * ts[0] * ts[1]), *caches))
    return (qp, qt[0], op, ot, Hq, kp, kt[0], vp, vt[0], okp, okt, Hkv, D, sp, pp, T, tp, ts[0],
            ts[1], 1 if interleaved else 0), out, (slots, positions)


def rotary_and_cache(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                     key_cache: torch.Tensor, value_cache: torch.Tensor,
                     slot_mapping: torch.Tensor, positions: torch.Tensor, table: torch.Tensor,
                     interleaved: bool = False, out: Optional[torch.Tensor] = None,
                     out_key: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turn ``query [T, Hq, D]`` and ``key [T, Hkv, D]`` by ``positions [T]``
    (int64) and write the turned keys and ``value [T, Hkv, D]`` to the cache as
    :func:`attention.reshape_and_cache_flash` does; returns the turned queries.

    The first ``table.size(1)`` dims of a row turn (:func:`rotary_table`): dims i
    and i + half of them, or with ``interleaved`` neighbours, are a pair; the
    others stay.  Computed in fp32 and rounded once.  A position outside the
    table gives NaN.  Token strides are free, the heads of a token dense.
    ``out`` (default: a new tensor) may be ``query`` itself, ``out_key``, which
    gets the turned keys (default: not kept), ``key``; neither may overlap anything
    else that the call takes.  All tokens of both are written, also those whose slot is
    skipped (negative or past the cache).  Of two
    tokens for one slot either may be left there, in parts."""
    _check_cache_view(key_cache, "key_cache")
    _check_cache_view(value_cache, "value_cache")
    dev = key_cache.device
    _check_on(value_cache, "value_cache", dev)
    shape, block_stride = key_cache.shape, key_cache.stride(0)
    if block_stride != value_cache.stride(0) or shape != value_cache.shape:
        raise ValueError("key_cache and value_cache must share shape and block stride")
    N, bs, Hkv, D = shape
    kp, vp = key_cache.data_ptr(), value_cache.data_ptr()
    nbytes = 2 * ((N - 1) * block_stride + bs * Hkv * D) if N else 0
    args, out, keep = _turn_args(query, key, value, slot_mapping, positions, table, interleaved,
                                 out, out_key, dev, True, (("key_cache", kp, kp + nbytes),
                                                           ("value_cache", vp, vp + nbytes)))
    dtype = query.dtype
    if key_cache.dtype != dtype or value_cache.dtype != dtype:
        raise ValueError("the rows and the caches must share one 16-bit dtype")
    if args[11] != Hkv or args[12] != D:
        raise ValueError("key/value must be [T, Hkv, D] matching the cache view")
    if args[15] == 0:
        return out
    with device_guard(dev):
        rc = _lib.load().aegkv_rotary_append(*args, kp, vp, block_stride, N, bs, _DTYPES[dtype],
                                             raw_stream(dev))
    _lib.check(rc, "rotary_and_cache")
    return out
