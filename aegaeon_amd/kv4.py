"""The KV cache held in 4 bits, beside the 16-bit one of :mod:`attention`:

* :func:`kv4_cache` — its storage, ``[N, L, Hkv, 2, 8.5 D]`` uint8, 3.76 times
  smaller; a block is opaque bytes to :mod:`ops` (swap, copy, pack, scatter,
  defrag) and to the block manager, as any other shape's;
* :func:`reshape_and_cache_kv4`, :func:`append_kv4` — the quantising write of
  new 16-bit K/V rows, one layer or every layer of a step;
* :func:`gather_tokens_kv4` — the de-page back to 16-bit rows;
* :func:`paged_decode_attention_kv4` — decode attention, one query token per
  sequence;
* :func:`varlen_attention_kv4` — attention of several query tokens per
  sequence: a prompt's next chunk over what is cached of it, or drafted tokens.

Values (include/aegkv.h has the bytes): 32 consecutive dims of a row share a
power of two, the rest of a value is its sign and one of 0, 0.5, 1, 1.5, 2, 3, 4,
6.  What is stored is exact in the rows' 16-bit type, which later calls on the
cache must pass as their own.  Everything is enqueued on the current torch
stream.
"""
from __future__ import annotations

from typing import Callable, Dict, Optional, Tuple

import torch

from . import _lib
from ._gpu import StreamBuffer, device_guard, raw_stream, stream_buffer
from .attention import (_DTYPES, _OWN_WORKSPACE, DecodePlan, _check_on, _check_rows, _gpu,
                        _int32_dense)

BLOCK_SIZE = 16


def kv4_record_bytes(head_dim: int) -> int:
    """Bytes of one kv head's K (or V) of a block: 4.25 bits per value."""
    if head_dim not in (64, 128, 256):
        raise ValueError("head_dim must be 64, 128 or 256")
    return 17 * head_dim // 2


def kv4_cache(n_blocks: int, n_layers: int, n_kv_heads: int, head_dim: int,
              device="cuda") -> torch.Tensor:
    """An empty cache ``[n_blocks, n_layers, n_kv_heads, 2, 8.5 head_dim]`` of
    uint8 (zeros: every value reads as 0)."""
    return torch.zeros((n_blocks, n_layers, n_kv_heads, 2, kv4_record_bytes(head_dim)),
                       dtype=torch.uint8, device=device)


def _check_cache(c: torch.Tensor, layers: bool, head_dim: int) -> None:
    """A cache ``[N, L, Hkv, 2, R]`` (one layer: ``[N, Hkv, 2, R]``) whose
    heads are dense; the block and layer strides are free."""
    shape, strides, r = c.shape, c.stride(), kv4_record_bytes(head_dim)
    names = "[N, L, Hkv, 2, R]" if layers else "[N, Hkv, 2, R]"
    if len(shape) != (5 if layers else 4) or not c.is_cuda or c.dtype != torch.uint8:
        raise ValueError(f"kv_cache must be a uint8 GPU tensor {names}")
    if shape[-1] != r or shape[-2] != 2:
        raise ValueError(f"kv_cache must be {names} with R = {r} bytes for head_dim {head_dim}")
    if strides[-1] != 1 or strides[-2] != r or strides[-3] != 2 * r:
        raise ValueError("kv_cache: each block must hold its heads' records densely")


def _check_new_rows(key: torch.Tensor, value: torch.Tensor, dim: int, names: str) -> None:
    if key.dim() != dim or value.shape != key.shape:
        raise ValueError(f"key and value must both be {names}")
    if key.dtype not in _DTYPES or value.dtype != key.dtype:
        raise ValueError("key and value must share a bf16/fp16 dtype")
    _check_rows(key, "key")
    _check_rows(value, "value")


def _check_slots(slot_mapping: torch.Tensor, tokens: int, device: torch.device) -> torch.Tensor:
    if slot_mapping.dtype != torch.int64 or not slot_mapping.is_cuda:
        raise ValueError("slot_mapping must be an int64 GPU tensor")
    _check_on(slot_mapping, "slot_mapping", device)
    if slot_mapping.dim() != 1 or slot_mapping.numel() < tokens:
        raise ValueError(f"slot_mapping must hold a slot for each of the {tokens} tokens")
    return slot_mapping.contiguous()


def reshape_and_cache_kv4(key: torch.Tensor, value: torch.Tensor, kv_cache: torch.Tensor,
                          slot_mapping: torch.Tensor) -> None:
    """Write rows ``key``/``value [T, Hkv, D]`` (dense rows, free token
    strides) into one layer ``kv_cache [N, Hkv, 2, R]`` of the 4-bit cache:
    row t goes to token ``s % 16`` of block ``s // 16``, ``s =
    slot_mapping[t]``; negative slots and slots past the cache are skipped.
    The slots must be distinct."""
    _check_new_rows(key, value, 3, "[T, Hkv, D]")
    _append(key.unsqueeze(0), value.unsqueeze(0), kv_cache.unsqueeze(1), slot_mapping,
            "reshape_and_cache_kv4")


def append_kv4(key: torch.Tensor, value: torch.Tensor, kv_cache: torch.Tensor,
               slot_mapping: torch.Tensor) -> None:
    """:func:`reshape_and_cache_kv4` for every layer in one launch:
    ``key``/``value [L, T, Hkv, D]`` (token and layer strides free) into
    ``kv_cache [N, L, Hkv, 2, R]``."""
    _check_new_rows(key, value, 4, "[L, T, Hkv, D]")
    _append(key, value, kv_cache, slot_mapping, "append_kv4")


def _append(key, value, kv_cache, slot_mapping, op: str) -> None:
    L, T, H, D = key.shape
    _check_cache(kv_cache, True, D)
    if kv_cache.size(1) != L or kv_cache.size(2) != H:
        raise ValueError("key/value and kv_cache disagree on the layers or kv heads")
    dev = kv_cache.device
    _check_on(key, "key", dev)
    _check_on(value, "value", dev)
    slots = _check_slots(slot_mapping, T, dev)
    if L == 0:
        return
    ks, vs, cs = key.stride(), value.stride(), kv_cache.stride()
    with device_guard(dev):
        rc = _lib.load().aegkv_kv4_append(
            key.data_ptr(), value.data_ptr(), ks[1], vs[1], ks[0] if L > 1 else 0,
            vs[0] if L > 1 else 0, slots.data_ptr(), T, kv_cache.data_ptr(), cs[0],
            cs[1] if L > 1 else 0, kv_cache.size(0), L, H, D, _DTYPES[key.dtype], raw_stream(dev))
    _lib.check(rc, op)


def gather_tokens_kv4(kv_cache: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                      total_tokens: int, max_seq_len: int, dtype: torch.dtype = torch.bfloat16,
                      layers: Optional[Tuple[int, int]] = None,
                      cu_seqlens: Optional[torch.Tensor] = None
                      ) -> Tuple[torch.Tensor, torch.Tensor]:
    """De-page sequences of ``kv_cache [N, L, Hkv, 2, R]``: returns ``(out_k,
    out_v)`` of shape ``[n_layers, total_tokens, Hkv, D]`` in ``dtype`` (the
    appended rows'), sequence b's tokens at ``cu_seqlens[b] : cu_seqlens[b] +
    seq_lens[b]``.  The other arguments are :func:`attention.gather_tokens`'s."""
    if dtype not in _DTYPES:
        raise ValueError("dtype must be bfloat16 or float16")
    if kv_cache.dim() != 5:
        raise ValueError("kv_cache must be a uint8 GPU tensor [N, L, Hkv, 2, R]")
    D = kv_cache.size(-1) * 2 // 17
    _check_cache(kv_cache, True, D)
    N, L, H = kv_cache.shape[:3]
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
    out_k = torch.empty((count, total_tokens, H, D), dtype=dtype, device=dev)
    out_v = torch.empty_like(out_k)
    if total_tokens == 0:
        return out_k, out_v
    with device_guard(dev):
        rc = _lib.load().aegkv_kv4_gather_tokens(
            kv_cache.data_ptr() + first * kv_cache.stride(1), kv_cache.stride(0),
            kv_cache.stride(1), N, bt.data_ptr(), bt.size(1), sl.data_ptr(),
            cu_seqlens.data_ptr(), sl.numel(), max_seq_len, out_k.data_ptr(), out_v.data_ptr(),
            total_tokens, total_tokens * H * D, count, H, D, _DTYPES[dtype], raw_stream(dev))
    _lib.check(rc, "gather_tokens_kv4")
    return out_k, out_v


def _check_cu(cu: torch.Tensor, name: str, batch: int, device: torch.device) -> None:
    _check_on(cu, name, device)
    if cu.dtype != torch.int32 or cu.dim() != 1 or not cu.is_contiguous() \
            or cu.numel() != batch + 1:
        raise ValueError(f"{name} must be a contiguous int32 GPU tensor [B + 1]")


# The workspaces of the calls that bring none, one per (device, stream).
_workspaces: Dict[Tuple[int, int], StreamBuffer] = {}


def _own_workspace(dev: torch.device, stream: int) -> Optional[StreamBuffer]:
    """The stream's shared workspace; None under graph capture, where a call
    takes memory of the graph's own pool instead: graphs captured on one stream
    may be replayed on several at once."""
    if torch.cuda.is_current_stream_capturing():
        return None
    return stream_buffer(_workspaces, dev, stream)


def paged_decode_attention_kv4(q: torch.Tensor, kv_cache: torch.Tensor,
                               block_tables: Optional[torch.Tensor],
                               seq_lens: Optional[torch.Tensor], scale: float, max_seq_len: int,
                               out: Optional[torch.Tensor] = None, n_workgroups: int = 0,
                               workspace: Optional[torch.Tensor] = None,
                               plan: Optional[DecodePlan] = None) -> torch.Tensor:
    """:func:`attention.paged_decode_attention` over one layer ``kv_cache
    [N, Hkv, 2, R]`` of the 4-bit cache (any block stride): ``q [B, Hq, D]`` ->
    ``out [B, Hq, D]``, both of the type the cache was written from.  Tables,
    lengths, ``n_workgroups``, ``plan`` (a :class:`attention.DecodePlan` serves
    either cache) and ``workspace`` (:func:`attention.attention_workspace`) are
    that function's; a sequence without tokens gives zeros.  ``scale``: any
    number that stays finite times log2 e.  New rows are appended by a call of
    their own, before this one."""
    return _paged_decode(_heads, "aegkv_kv4_decode_attention", "paged_decode_attention_kv4", q,
                         kv_cache, block_tables, seq_lens, scale, max_seq_len, out, n_workgroups,
                         workspace, plan)


def _heads(c: torch.Tensor, head_dim: int) -> int:
    """The kv heads of one layer ``[N, Hkv, 2, R]``."""
    _check_cache(c, False, head_dim)
    return c.size(1)


def _paged_decode(heads_of: Callable[[torch.Tensor, int], int], entry: str, op: str,
                  q: torch.Tensor, kv_cache: torch.Tensor, block_tables: Optional[torch.Tensor],
                  seq_lens: Optional[torch.Tensor], scale: float, max_seq_len: int,
                  out: Optional[torch.Tensor], n_workgroups: int,
                  workspace: Optional[torch.Tensor], plan: Optional[DecodePlan]) -> torch.Tensor:
    """Decode attention over one layer of a 4- or 8-bit cache: ``heads_of``
    checks the cache and tells its kv heads, ``entry`` names the C entry."""
    shape, q_strides, dev = q.shape, q.stride(), q.device
    if len(shape) != 3 or q_strides[2] != 1 or q_strides[1] != shape[2] or not q.is_cuda:
        raise ValueError("q must be a GPU tensor [B, Hq, D] with dense heads")
    dtype = _DTYPES.get(q.dtype)
    if dtype is None:
        raise ValueError("q must be bf16 or fp16")
    B, Hq, D = shape
    Hkv = heads_of(kv_cache, D)
    if kv_cache.device != dev:
        raise ValueError(f"kv_cache must be a GPU tensor on {dev} (got {kv_cache.device})")
    if plan is not None:  # whose tables and lengths were checked when it was built
        if plan.buffer.device != dev:
            raise ValueError(f"the plan lives on {plan.buffer.device}, the call on {dev}")
        for given, held, name in ((block_tables, plan.block_tables, "block_tables"),
                                  (seq_lens, plan.seq_lens, "seq_lens")):
            if given is not None and given.data_ptr() != held.data_ptr():
                raise ValueError(f"{name} is not the tensor the plan was built from")
        if max_seq_len != plan.max_seq_len or n_workgroups != plan.n_workgroups \
                or B != plan.batch or Hkv != plan.n_kv_heads:
            raise ValueError("the plan was built for another batch, max_seq_len, kv-head count "
                             "or workgroup count")
        sl = plan.seq_lens
    else:
        if block_tables is None or seq_lens is None:
            raise ValueError("block_tables and seq_lens are required without a plan")
        _check_on(block_tables, "block_tables", dev)
        _check_on(seq_lens, "seq_lens", dev)
        if block_tables.dim() != 2 or seq_lens.dim() != 1 or block_tables.size(0) != B \
                or seq_lens.numel() != B:
            raise ValueError("block_tables must be [B, max_blocks] and seq_lens [B] for q's batch")
        sl = _int32_dense(seq_lens)
    out = _check_out(out, q)
    if B == 0:
        return out
    lib = _lib.load()
    with device_guard(dev):
        ws_bytes = lib.aegkv_paged_decode_attention_workspace_size(B, Hq, Hkv, D, max_seq_len,
                                                                   dtype, n_workgroups)
        if ws_bytes < 0:
            _lib.check(int(ws_bytes), "attention_workspace_bytes")
        stream = raw_stream(dev)
        shared = _own_workspace(dev, stream) if workspace is None else None
        if workspace is not None:
            _check_workspace(workspace, ws_bytes, dev)
        args = (out.data_ptr(), out.stride(0), q.data_ptr(), q_strides[0], kv_cache.data_ptr(),
                kv_cache.stride(0), kv_cache.size(0))
        if plan is not None:
            if stream != plan.raw_stream:
                plan.wait_for_build(torch.cuda.current_stream(dev))
            args += (plan.buffer.data_ptr(), plan.nbytes)
            call = getattr(lib, entry + "_planned")
        else:
            bt = _int32_dense(block_tables)
            args += (bt.data_ptr(), bt.size(1))
            call = getattr(lib, entry)
        with _OWN_WORKSPACE if shared is None else shared.lock:
            if shared is not None:
                workspace = shared.at_least(ws_bytes, dev)
            elif workspace is None:
                workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
            rc = call(*args, sl.data_ptr(), B, max_seq_len, Hq, Hkv, D, float(scale), dtype,
                      n_workgroups, workspace.data_ptr(), ws_bytes, stream)
    _lib.check(rc, op)
    return out


def _check_out(out: Optional[torch.Tensor], q: torch.Tensor) -> torch.Tensor:
    if out is None:
        return q.new_empty(q.shape)
    if out.shape != q.shape or out.stride(2) != 1 or out.stride(1) != q.size(2):
        raise ValueError("out must have q's shape, with dense heads")
    if out.dtype != q.dtype:
        raise ValueError("out must have q's dtype")
    _check_on(out, "out", q.device)
    return out


def _check_workspace(workspace: torch.Tensor, nbytes: int, dev: torch.device) -> None:
    _check_on(workspace, "workspace", dev)
    if not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < nbytes:
        raise ValueError(f"workspace holds {workspace.numel() * workspace.element_size()} bytes, "
                         f"the call needs {nbytes} in one piece")


def varlen_attention_kv4(q: torch.Tensor, kv_cache: torch.Tensor, block_tables: torch.Tensor,
                         cu_seqlens_q: torch.Tensor, seq_lens: torch.Tensor, max_seqlen_q: int,
                         max_seq_len: int, scale: float, causal: bool = True,
                         out: Optional[torch.Tensor] = None,
                         workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of several query tokens per sequence over one layer
    ``kv_cache [N, Hkv, 2, R]`` of the 4-bit cache: ``q [T, Hq, D]`` (any token
    stride, dense heads) -> ``out [T, Hq, D]``, both of the type the cache was
    written from.  Sequence b's queries are ``cu_seqlens_q[b] ..
    cu_seqlens_q[b + 1]`` (int32 on the GPU), the last of its ``seq_lens[b]``
    cached tokens (append them first); query i of m attends to keys ``j <=
    seq_lens[b] - m + i``, all of them when not ``causal``, and gives zeros
    without any.  ``max_seqlen_q`` and ``max_seq_len`` are host bounds: queries
    past the first are left alone, keys past the second not attended.  head_dim
    64 or 128.  ``workspace``: :func:`varlen_attention_workspace` (reusable on
    one stream, by one thread at a time); by default one per (device, stream)
    that threads may share."""
    return _varlen(_heads, "aegkv_kv4_varlen_attention", "varlen_attention_kv4", q, kv_cache,
                   block_tables, cu_seqlens_q, seq_lens, max_seqlen_q, max_seq_len, scale, causal,
                   out, workspace)


def _varlen(heads_of: Callable[[torch.Tensor, int], int], entry: str, op: str, q: torch.Tensor,
            kv_cache: torch.Tensor, block_tables: torch.Tensor, cu_seqlens_q: torch.Tensor,
            seq_lens: torch.Tensor, max_seqlen_q: int, max_seq_len: int, scale: float,
            causal: bool, out: Optional[torch.Tensor],
            workspace: Optional[torch.Tensor]) -> torch.Tensor:
    """Attention of several query tokens per sequence over one layer of a 4- or
    8-bit cache (see :func:`_paged_decode`)."""
    if q.dim() != 3:
        raise ValueError("q must be [tokens, Hq, D]")
    _check_rows(q, "q")
    if q.dtype not in _DTYPES:
        raise ValueError("q must be bf16 or fp16")
    T, Hq, D = q.shape
    dev = q.device
    Hkv = heads_of(kv_cache, D)
    _check_on(kv_cache, "kv_cache", dev)
    _check_on(block_tables, "block_tables", dev)
    _check_on(seq_lens, "seq_lens", dev)
    B = seq_lens.numel()
    if block_tables.dim() != 2 or seq_lens.dim() != 1 or block_tables.size(0) != B:
        raise ValueError("block_tables must be [B, max_blocks] and seq_lens [B]")
    _check_cu(cu_seqlens_q, "cu_seqlens_q", B, dev)
    out = _check_out(out, q)
    if B == 0 or T == 0:
        return out
    bt, sl = _int32_dense(block_tables), _int32_dense(seq_lens)
    lib = _lib.load()
    sizes = (int(max_seqlen_q), int(max_seq_len), Hq, Hkv, D)
    dtype = _DTYPES[q.dtype]
    with device_guard(dev):
        ws_bytes = getattr(lib, entry + "_workspace_size")(B, T, *sizes, dtype)
        if ws_bytes < 0:
            _lib.check(int(ws_bytes), "varlen_attention_workspace")
        stream = raw_stream(dev)
        shared = None
        if workspace is not None:
            _check_workspace(workspace, ws_bytes, dev)
        elif ws_bytes > 0:
            shared = _own_workspace(dev, stream)
        with _OWN_WORKSPACE if shared is None else shared.lock:
            if shared is not None:
                workspace = shared.at_least(ws_bytes, dev)
            elif workspace is None and ws_bytes > 0:
                workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
            rc = getattr(lib, entry)(
                out.data_ptr(), out.stride(0), q.data_ptr(), q.stride(0), kv_cache.data_ptr(),
                kv_cache.stride(0), kv_cache.size(0), bt.data_ptr(), bt.size(1),
                cu_seqlens_q.data_ptr(), sl.data_ptr(), B, T, *sizes, float(scale),
                int(bool(causal)), dtype, workspace.data_ptr() if ws_bytes > 0 else None, ws_bytes,
                stream)
    _lib.check(rc, op)
    return out


def varlen_attention_workspace(batch: int, total_q: int, max_seqlen_q: int, max_seq_len: int,
                               n_q_heads: int, n_kv_heads: int, head_dim: int,
                               dtype: torch.dtype = torch.bfloat16,
                               device=None) -> Optional[torch.Tensor]:
    """A workspace for :func:`varlen_attention_kv4` calls of exactly these
    sizes on ``device`` (None when they need none)."""
    return _varlen_workspace("aegkv_kv4_varlen_attention", batch, total_q, max_seqlen_q,
                             max_seq_len, n_q_heads, n_kv_heads, head_dim, dtype, device)


def _varlen_workspace(entry: str, batch: int, total_q: int, max_seqlen_q: int, max_seq_len: int,
                      n_q_heads: int, n_kv_heads: int, head_dim: int, dtype: torch.dtype,
                      device) -> Optional[torch.Tensor]:
    if dtype not in _DTYPES:
        raise ValueError("dtype must be bfloat16 or float16")
    dev = _gpu(device)
    with device_guard(dev):
        n = getattr(_lib.load(), entry + "_workspace_size")(
            batch, total_q, max_seqlen_q, max_seq_len, n_q_heads, n_kv_heads, head_dim,
            _DTYPES[dtype])
    if n < 0:
        _lib.check(int(n), "varlen_attention_workspace")
    return torch.empty(int(n), dtype=torch.uint8, device=dev) if n > 0 else None
