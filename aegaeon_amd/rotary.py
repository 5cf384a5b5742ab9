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

from typing import Optional

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


def _check_table(table: torch.Tensor, head_dim: int, dev: torch.device) -> None:
    _check_on(table, "table", dev)
    if table.dtype != torch.float32 or table.dim() != 2 or not table.is_contiguous():
        raise ValueError("table must be a contiguous float32 tensor [positions, rotary_dim]")
    if table.size(0) == 0 or table.size(1) == 0 or table.size(1) > head_dim:
        raise ValueError(f"table must have rows of up to head_dim {head_dim} entries")


def _check_token_ids(x: torch.Tensor, name: str, tokens: int, dev: torch.device) -> torch.Tensor:
    _check_on(x, name, dev)
    if x.dtype != torch.int64 or x.dim() != 1 or x.numel() < tokens:
        raise ValueError(f"{name} must be an int64 GPU tensor with an entry for each of the "
                         f"{tokens} tokens")
    return x.contiguous()


def _check_like(t: torch.Tensor, x: torch.Tensor, name: str) -> torch.Tensor:
    if t.shape != x.shape or t.dtype != x.dtype:
        raise ValueError(f"{name} must have the shape and dtype {tuple(x.shape)}, {x.dtype}")
    _check_rows(t, name)
    _check_on(t, name, x.device)
    return t


def _span(t: torch.Tensor):
    """First byte and the byte past the last of rows ``[T, H, D]``."""
    first = t.data_ptr()
    return first, first + ((t.size(0) - 1) * t.stride(0) + t.size(1) * t.size(2)) * 2


def _check_apart(t: torch.Tensor, x: torch.Tensor, name: str, of: str, same: bool) -> None:
    """``t``, written, may be ``x``, read (``same``), or must not share bytes
    with it."""
    if same and t.data_ptr() == x.data_ptr() and t.stride() == x.stride():
        return
    (a, b), (c, d) = _span(t), _span(x)
    # rows of one wider buffer (the slices of a fused projection) interleave
    if a < d and c < b and not (t.stride(0) == x.stride(0) and _columns_apart(t, x)):
        raise ValueError(f"{name} overlaps {of}")


def _columns_apart(t: torch.Tensor, x: torch.Tensor) -> bool:
    step = t.stride(0) * 2
    if step == 0:
        return False
    off = (x.data_ptr() - t.data_ptr()) % step
    return off >= t.size(1) * t.size(2) * 2 and off + x.size(1) * x.size(2) * 2 <= step


def _check_turned(query, key, value, slot_mapping, positions, table, out, out_key, dev,
                  key_in_place: bool):
    """The arguments that both caches' calls share; (slots, positions, out)."""
    for x, n in ((query, "query"), (key, "key"), (value, "value")):
        if x.dim() != 3:
            raise ValueError(f"{n} must be [tokens, heads, head_dim]")
        _check_rows(x, n)
        _check_on(x, n, dev)
    T, _, D = query.shape
    if key.size(0) != T or key.size(2) != D or value.shape != key.shape:
        raise ValueError("key and value must be [T, Hkv, D] with query's tokens and head_dim")
    if query.dtype not in _DTYPES or key.dtype != query.dtype or value.dtype != query.dtype:
        raise ValueError("query, key and value must share a bf16/fp16 dtype")
    _check_table(table, D, dev)
    slots = _check_token_ids(slot_mapping, "slot_mapping", T, dev)
    positions = _check_token_ids(positions, "positions", T, dev)
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=dev)
    elif T > 0:
        _check_like(out, query, "out")
        _check_apart(out, query, "out", "query", True)
        _check_apart(out, key, "out", "key", False)
        _check_apart(out, value, "out", "value", False)
    if out_key is not None and T > 0:
        _check_like(out_key, key, "out_key")
        _check_apart(out_key, key, "out_key", "key", key_in_place)
        _check_apart(out_key, query, "out_key", "query", False)
        _check_apart(out_key, value, "out_key", "value", False)
        _check_apart(out_key, out, "out_key", "out", False)
    return slots, positions, out


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
