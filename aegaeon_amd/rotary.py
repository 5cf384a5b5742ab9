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


def _check_like(t: torch.Tensor, x: torch.Tensor, name: str) -> torch.Tensor:
    if t.shape != x.shape or t.dtype != x.dtype:
        raise ValueError(f"{name} must have the shape and dtype {tuple(x.shape)}, {x.dtype}")
    _check_rows(t, name)
    _check_on(t, name, x.device)
    return t


def _span(t: torch.Tensor):
    """First byte, the byte past the last and the token stride in bytes of rows
    ``[T, H, D]``."""
    T, H, D = t.shape
    first, step = t.data_ptr(), 2 * t.stride(0)
    return first, first + (T - 1) * step + 2 * H * D, step, 2 * H * D


def _check_apart(name: str, written, read, same: Tuple[str, ...]) -> None:
    """``written``, a span, may be one of ``read``'s spans that ``same`` names,
    and shares no byte with the others."""
    a, b, step, row = written
    for of, (c, d, other_step, other_row) in read.items():
        if a >= d or c >= b or (of in same and a == c and step == other_step):
            continue
        # slices of one wider buffer (a fused projection's columns) lie side by side
        if step == other_step and step > 0:
            off = (c - a) % step
            if off >= row and off + other_row <= step:
                continue
        raise ValueError(f"{name} overlaps {of}")


def _check_turned(query, key, value, slot_mapping, positions, table, out, out_key, dev,
                  key_in_place: bool):
    """The arguments that both caches' calls share; (slots, positions, out)."""
    qs, ks, dtype = query.shape, key.shape, query.dtype
    if len(qs) != 3 or len(ks) != 3 or value.shape != ks or ks[0] != qs[0] or ks[2] != qs[2]:
        raise ValueError("query must be [T, Hq, D], key and value [T, Hkv, D] with its tokens "
                         "and head_dim")
    if dtype not in _DTYPES or key.dtype != dtype or value.dtype != dtype:
        raise ValueError("query, key and value must share a bf16/fp16 dtype")
    T, _, D = qs
    index = dev.index
    for x, n in ((query, "query"), (key, "key"), (value, "value")):
        strides = x.stride()
        if x.get_device() != index or strides[2] != 1 or strides[1] != D:
            _check_on(x, n, dev)
            _check_rows(x, n)
    for x, n in ((slot_mapping, "slot_mapping"), (positions, "positions")):
        if x.get_device() != index:
            _check_on(x, n, dev)
        if x.dtype != torch.int64 or x.dim() != 1 or x.numel() < T:
            raise ValueError(f"{n} must be an int64 GPU tensor with an entry for each of the {T} "
                             "tokens")
    if table.get_device() != index:
        _check_on(table, "table", dev)
    ts = table.shape
    if table.dtype != torch.float32 or len(ts) != 2 or not table.is_contiguous() or ts[0] == 0 \
            or not 0 < ts[1] <= D:
        raise ValueError("table must be a contiguous float32 tensor [positions, rotary_dim] with "
                         f"rows of up to head_dim {D} entries")
    if T > 0 and (out is not None or out_key is not None):
        read = {"query": _span(query), "key": _span(key), "value": _span(value)}
        if out is not None:
            written = _span(_check_like(out, query, "out"))
            _check_apart("out", written, read, ("query",))
            read["out"] = written
        if out_key is not None:
            _check_apart("out_key", _span(_check_like(out_key, key, "out_key")), read,
                         ("key",) if key_in_place else ())
    return slot_mapping.contiguous(), positions.contiguous(), \
        query.new_empty(qs) if out is None else out


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
    gets the turned keys (default: not kept), ``key``; all tokens of both are
    written, also those whose slot is skipped (negative or past the cache)."""
    _check_cache_view(key_cache, "key_cache")
    _check_cache_view(value_cache, "value_cache")
    dev = key_cache.device
    _check_on(value_cache, "value_cache", dev)
    slots, positions, out = _check_turned(query, key, value, slot_mapping, positions, table, out,
                                          out_key, dev, True)
    if key_cache.stride(0) != value_cache.stride(0) or key_cache.shape != value_cache.shape:
        raise ValueError("key_cache and value_cache must share shape and block stride")
    if key_cache.dtype != key.dtype or value_cache.dtype != key.dtype:
        raise ValueError("the rows and the caches must share one 16-bit dtype")
    if key.shape[1:] != key_cache.shape[2:]:
        raise ValueError("key/value must be [T, Hkv, D] matching the cache view")
    T, Hq, D = query.shape
    if T == 0:
        return out
    N, bs, Hkv, _ = key_cache.shape
    with device_guard(dev):
        rc = _lib.load().aegkv_rotary_append(
            query.data_ptr(), query.stride(0), out.data_ptr(), out.stride(0), Hq, key.data_ptr(),
            key.stride(0), value.data_ptr(), value.stride(0),
            None if out_key is None else out_key.data_ptr(),
            0 if out_key is None else out_key.stride(0), Hkv, D, slots.data_ptr(),
            positions.data_ptr(), T, table.data_ptr(), table.size(0), table.size(1),
            int(bool(interleaved)), key_cache.data_ptr(), value_cache.data_ptr(),
            key_cache.stride(0), N, bs, _DTYPES[query.dtype], raw_stream(dev))
    _lib.check(rc, "rotary_and_cache")
    return out
