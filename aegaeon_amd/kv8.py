"""The KV cache held in 8 bits, beside the 16-bit one of :mod:`attention` and the
4-bit one of :mod:`kv4`:

* :func:`kv8_cache` — its storage, ``[N, L, R]`` uint8, R = 32 Hkv D bytes of
  codes and a line of scales: half the 16-bit cache's; a block is opaque bytes to
  :mod:`ops` (swap, copy, pack, scatter, defrag) and to the block manager, as any
  other shape's;
* :func:`reshape_and_cache_kv8`, :func:`append_kv8` — the quantising write of new
  16-bit K/V rows, one layer or every layer of a step;
* :func:`rotary_and_cache_kv8` — the same for one layer with keys and queries
  turned by their positions on the way;
* :func:`gather_tokens_kv8` — the de-page back to 16-bit rows;
* :func:`paged_decode_attention_kv8` — decode attention, one query token per
  sequence;
* :func:`varlen_attention_kv8` — attention of several query tokens per sequence: a
  prompt's next chunk over what is cached of it, or drafted tokens.

Values (include/aegkv.h has the bytes): the 16 tokens of a block share a power of
two per head and side (K or V), the rest of a value is an 8-bit float of three
mantissa bits.  What is stored is exact in the rows' 16-bit type, which later
calls on the cache must pass as their own.  Everything is enqueued on the current
torch stream.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._gpu import device_guard, raw_stream
from .attention import _DTYPES, DecodePlan, _check_on, _int32_dense
from .kv4 import (_check_cu, _check_new_rows, _check_slots, _paged_decode, _varlen,
                  _varlen_workspace)
from .rotary import _turn_args

BLOCK_SIZE = 16
MAX_KV_HEADS = 256


def kv8_block_bytes(n_kv_heads: int, head_dim: int) -> int:
    """Bytes of a layer's block: a byte per value, 4 per kv head, whole lines."""
    if head_dim not in (64, 128, 256):
        raise ValueError("head_dim must be 64, 128 or 256")
    if not 0 < n_kv_heads <= MAX_KV_HEADS:
        raise ValueError(f"n_kv_heads must be 1 to {MAX_KV_HEADS}")
    return 32 * n_kv_heads * head_dim + -(-4 * n_kv_heads // 128) * 128


def kv8_cache(n_blocks: int, n_layers: int, n_kv_heads: int, head_dim: int,
              device="cuda") -> torch.Tensor:
    """An empty cache ``[n_blocks, n_layers, kv8_block_bytes]`` of uint8 (zeros:
    every value reads as 0)."""
    return torch.zeros((n_blocks, n_layers, kv8_block_bytes(n_kv_heads, head_dim)),
                       dtype=torch.uint8, device=device)


def _kv_heads(c: torch.Tensor, layers: bool, head_dim: int) -> int:
    """The kv heads of a cache ``[N, L, R]`` (one layer: ``[N, R]``) of
    ``head_dim``; its block and layer strides are free."""
    shape = c.shape
    names = "[N, L, R]" if layers else "[N, R]"
    if len(shape) != (3 if layers else 2) or not c.is_cuda or c.dtype != torch.uint8:
        raise ValueError(f"kv_cache must be a uint8 GPU tensor {names}")
    if head_dim not in (64, 128, 256):
        raise ValueError("head_dim must be 64, 128 or 256")
    heads = shape[-1] // (32 * head_dim)
    if not 0 < heads <= MAX_KV_HEADS or shape[-1] != kv8_block_bytes(heads, head_dim):
        raise ValueError(f"kv_cache must be {names} with R = kv8_block_bytes(n_kv_heads, "
                         f"{head_dim}) bytes (got {shape[-1]})")
    if c.stride(-1) != 1:
        raise ValueError("kv_cache: each layer's block must be dense")
    return heads


def reshape_and_cache_kv8(key: torch.Tensor, value: torch.Tensor, kv_cache: torch.Tensor,
                          slot_mapping: torch.Tensor) -> None:
    """Write rows ``key``/``value [T, Hkv, D]`` (dense rows, free token strides)
    into one layer ``kv_cache [N, R]`` of the 8-bit cache: row t goes to token
    ``s % 16`` of block ``s // 16``, ``s = slot_mapping[t]``; negative slots and
    slots past the cache are skipped.  A row at a block's first token begins the
    block anew; others join what it holds, whose values are rounded once more
    where their size raises the block's exponent.  The rows of one block must
    follow each other in the call (skipped ones may lie between them, another block's
    not: the block's values may be wrong then); of several for one slot the last
    counts."""
    _check_new_rows(key, value, 3, "[T, Hkv, D]")
    _append(key, value, kv_cache, slot_mapping, False, "reshape_and_cache_kv8")


def append_kv8(key: torch.Tensor, value: torch.Tensor, kv_cache: torch.Tensor,
               slot_mapping: torch.Tensor) -> None:
    """:func:`reshape_and_cache_kv8` for every layer in one launch:
    ``key``/``value [L, T, Hkv, D]`` (token and layer strides free) into
    ``kv_cache [N, L, R]``."""
    _check_new_rows(key, value, 4, "[L, T, Hkv, D]")
    _append(key, value, kv_cache, slot_mapping, True, "append_kv8")


def _append(key, value, kv_cache, slot_mapping, layers: bool, op: str) -> None:
    T, H, D = key.shape[-3:]
    L = key.size(0) if layers else 1
    if _kv_heads(kv_cache, layers, D) != H or (layers and kv_cache.size(1) != L):
        raise ValueError("key/value and kv_cache disagree on the layers or kv heads")
    dev = kv_cache.device
    _check_on(key, "key", dev)
    _check_on(value, "value", dev)
    slots = _check_slots(slot_mapping, T, dev)
    if L == 0 or T == 0:
        return
    ks, vs, cs = key.stride(), value.stride(), kv_cache.stride()
    k_layer, v_layer, c_layer = (ks[0], vs[0], cs[1]) if L > 1 else (0, 0, 0)
    with device_guard(dev):
        rc = _lib.load().aegkv_kv8_append(
            key.data_ptr(), value.data_ptr(), ks[-3], vs[-3], k_layer, v_layer, slots.data_ptr(), T,
            kv_cache.data_ptr(), cs[0], c_layer, kv_cache.size(0), L, H, D, _DTYPES[key.dtype],
            raw_stream(dev))
    _lib.check(rc, op)


def rotary_and_cache_kv8(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                         kv_cache: torch.Tensor, slot_mapping: torch.Tensor,
                         positions: torch.Tensor, table: torch.Tensor, interleaved: bool = False,
                         out: Optional[torch.Tensor] = None,
                         out_key: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`rotary.rotary_and_cache` into one layer ``kv_cache [N, R]`` of the
    8-bit cache, with :func:`reshape_and_cache_kv8`'s slots and blocks: returns the
    turned queries.  The codes are those of the turned keys in fp32, without a
    rounding to 16 bits between; ``out_key``, in 16 bits, must not be ``key``."""
    if query.dim() == 0:
        raise ValueError("query must be [T, Hq, D]")
    dev, heads = kv_cache.device, _kv_heads(kv_cache, False, query.shape[-1])
    N, R = kv_cache.shape
    cp, block_stride = kv_cache.data_ptr(), kv_cache.stride(0)
    args, out, keep = _turn_args(query, key, value, slot_mapping, positions, table, interleaved,
                                 out, out_key, dev, False,
                                 (("kv_cache", cp, cp + ((N - 1) * block_stride + R if N else 0)),))
    if heads != args[11]:
        raise ValueError("key/value and kv_cache disagree on the kv heads")
    if args[15] == 0:
        return out
    with device_guard(dev):
        rc = _lib.load().aegkv_kv8_rotary_append(*args, cp, block_stride, N, _DTYPES[query.dtype],
                                                 raw_stream(dev))
    _lib.check(rc, "rotary_and_cache_kv8")
    return out


def gather_tokens_kv8(kv_cache: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                      total_tokens: int, max_seq_len: int, head_dim: int,
                      dtype: torch.dtype = torch.bfloat16,
                      layers: Optional[Tuple[int, int]] = None,
                      cu_seqlens: Optional[torch.Tensor] = None
                      ) -> Tuple[torch.Tensor, torch.Tensor]:
    """De-page sequences of ``kv_cache [N, L, R]``: returns ``(out_k, out_v)`` of
    shape ``[n_layers, total_tokens, Hkv, head_dim]`` in ``dtype`` (the appended
    rows'), sequence b's tokens at ``cu_seqlens[b] : cu_seqlens[b] +
    seq_lens[b]``.  The other arguments are :func:`attention.gather_tokens`'s."""
    if dtype not in _DTYPES:
        raise ValueError("dtype must be bfloat16 or float16")
    H = _kv_heads(kv_cache, True, head_dim)
    N, L = kv_cache.shape[:2]
    first, count = layers if layers is not None else (0, L)
    if not (0 <= first and first + count <= L and count > 0):
        raise ValueError("layer range out of bounds")
    dev = kv_cache.device
    _check_on(block_tables, "block_tables", dev)
    _check_on(seq_lens, "seq_lens", dev)
    if block_tables.dim() != 2 or seq_lens.dim() != 1 or block_tables.size(0) != seq_lens.numel():
        raise ValueError("block_tables must be [B, max_blocks] and seq_lens [B]")
    bt = _int32_dense(block_tables)
    sl = _int32_dense(seq_lens)
    if cu_seqlens is None:
        cu_seqlens = torch.zeros(sl.numel() + 1, dtype=torch.int32, device=dev)
        torch.cumsum(sl, 0, dtype=torch.int32, out=cu_seqlens[1:])
    else:
        _check_cu(cu_seqlens, "cu_seqlens", sl.numel(), dev)
    # (views of one allocation: a microsecond less of the host)
    out_k, out_v = torch.empty((2, count, total_tokens, H, head_dim), dtype=dtype,
                               device=dev).unbind(0)
    if total_tokens == 0:
        return out_k, out_v
    with device_guard(dev):
        rc = _lib.load().aegkv_kv8_gather_tokens(
            kv_cache.data_ptr() + first * kv_cache.stride(1), kv_cache.stride(0),
            kv_cache.stride(1), N, bt.data_ptr(), bt.size(1), sl.data_ptr(),
            cu_seqlens.data_ptr(), sl.numel(), max_seq_len, out_k.data_ptr(), out_v.data_ptr(),
            total_tokens, total_tokens * H * head_dim, count, H, head_dim, _DTYPES[dtype],
            raw_stream(dev))
    _lib.check(rc, "gather_tokens_kv8")
    return out_k, out_v


def _layer_heads(c: torch.Tensor, head_dim: int) -> int:
    return _kv_heads(c, False, head_dim)


def paged_decode_attention_kv8(q: torch.Tensor, kv_cache: torch.Tensor,
                               block_tables: Optional[torch.Tensor],
                               seq_lens: Optional[torch.Tensor], scale: float, max_seq_len: int,
                               out: Optional[torch.Tensor] = None, n_workgroups: int = 0,
                               workspace: Optional[torch.Tensor] = None,
                               plan: Optional[DecodePlan] = None) -> torch.Tensor:
    """:func:`attention.paged_decode_attention` over one layer ``kv_cache
    [N, R]`` of the 8-bit cache (any block stride): ``q [B, Hq, D]`` -> ``out
    [B, Hq, D]``, both of the type the cache was written from.  Tables, lengths,
    ``n_workgroups``, ``plan`` (a :class:`attention.DecodePlan` serves any of the
    caches) and ``workspace`` (:func:`attention.attention_workspace`) are that
    function's; a sequence without tokens gives zeros.  ``scale``: any number that
    stays finite times log2 e.  New rows are appended by a call of their own,
    before this one."""
    return _paged_decode(_layer_heads, "aegkv_kv8_decode_attention", "paged_decode_attention_kv8",
                         q, kv_cache, block_tables, seq_lens, scale, max_seq_len, out,
                         n_workgroups, workspace, plan)


def varlen_attention_kv8(q: torch.Tensor, kv_cache: torch.Tensor, block_tables: torch.Tensor,
                         cu_seqlens_q: torch.Tensor, seq_lens: torch.Tensor, max_seqlen_q: int,
                         max_seq_len: int, scale: float, causal: bool = True,
                         out: Optional[torch.Tensor] = None,
                         workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`kv4.varlen_attention_kv4` over one layer ``kv_cache [N, R]`` of the
    8-bit cache: ``q [T, Hq, D]`` (any token stride, dense heads) -> ``out [T, Hq,
    D]``, both of the type the cache was written from.  Sequence b's queries are
    ``cu_seqlens_q[b] .. cu_seqlens_q[b + 1]`` (int32 on the GPU), the last of its
    ``seq_lens[b]`` cached tokens (append them first); query i of m attends to keys
    ``j <= seq_lens[b] - m + i``, all of them when not ``causal``, and gives zeros
    without any.  ``max_seqlen_q`` and ``max_seq_len`` are host bounds: queries past
    the first are left alone, keys past the second not attended.  head_dim 64 or
    128.  ``workspace``: :func:`varlen_attention_workspace` (reusable on one stream,
    by one thread at a time); by default one per (device, stream) that threads may
    share."""
    return _varlen(_layer_heads, "aegkv_kv8_varlen_attention", "varlen_attention_kv8", q, kv_cache,
                   block_tables, cu_seqlens_q, seq_lens, max_seqlen_q, max_seq_len, scale, causal,
                   out, workspace)


def varlen_attention_workspace(batch: int, total_q: int, max_seqlen_q: int, max_seq_len: int,
                               n_q_heads: int, n_kv_heads: int, head_dim: int,
                               dtype: torch.dtype = torch.bfloat16,
                               device=None) -> Optional[torch.Tensor]:
    """A workspace for :func:`varlen_attention_kv8` calls of exactly these sizes
    on ``device`` (None when they need none)."""
    return _varlen_workspace("aegkv_kv8_varlen_attention", batch, total_q, max_seqlen_q,
                             max_seq_len, n_q_heads, n_kv_heads, head_dim, dtype, device)
