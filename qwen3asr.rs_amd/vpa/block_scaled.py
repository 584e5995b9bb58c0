"""A paged cache of E4M3 bytes with one scale per block and kv head: the append that
sets the scales (``vpa_reshape_and_cache_block_scaled``) and the attention that reads them
(``vpa_paged_attention_block_scaled``)."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import VpaError, check
from .ops import _err, _on_device_of, _ptr, _same_device, _stream, cache_geometry, dtype_code


def block_scales(num_blocks: int, num_kv_heads: int, device) -> Tuple[torch.Tensor, torch.Tensor]:
    """Scales f32 [num_blocks, num_kv_heads] for a pool's K and V (zeros: nothing written)."""
    return (torch.zeros((num_blocks, num_kv_heads), device=device),
            torch.zeros((num_blocks, num_kv_heads), device=device))


def _geometry(key_cache, value_cache, key_scales, value_scales):
    """``cache_geometry`` of an fp8 cache and the scales' block stride. (Called for every
    layer of a step: one look at each shape and stride, the messages where one is wrong.)"""
    kd, vd = key_cache.dtype, value_cache.dtype
    if kd is vd and (kd is torch.float8_e4m3fn or kd is torch.uint8) and key_cache.dim() == 5 \
            and value_cache.dim() == 4:
        nb, kvh, dx, bs, x = key_cache.shape
        s0, s1, s2, s3, s4 = key_cache.stride()
        d = dx * 16
        if x == 16 and value_cache.shape == (nb, kvh, d, bs) and s4 == 1 and s3 == 16 and \
                s2 == bs * 16 and value_cache.stride() == (s0, s1, bs, 1) and s1 >= d * bs and \
                key_scales.dtype is value_scales.dtype is torch.float32 and \
                key_scales.shape == value_scales.shape == (nb, kvh):
            stride = key_scales.stride()
            if value_scales.stride() == stride and stride[1] == 1 and nb > 1:
                return nb, kvh, d, bs, s0, s1, stride[0]
    geometry = cache_geometry(key_cache, value_cache)
    nb, kvh = geometry[:2]
    if dtype_code(key_cache.dtype) != _lib.DTYPE_FP8_E4M3:
        raise VpaError(_lib.VPA_ERR_UNSUPPORTED,
                       f"a block-scaled cache is fp8 (E4M3 bytes), got {key_cache.dtype}")
    for name, t in (("key_scales", key_scales), ("value_scales", value_scales)):
        if t.dtype != torch.float32 or t.shape != (nb, kvh) or (kvh > 1 and t.stride(1) != 1):
            raise _err(f"{name} must be f32 [{nb}, {kvh}] with contiguous heads, got {t.dtype} "
                       f"{tuple(t.shape)}")
    stride = key_scales.stride(0) if nb > 1 else kvh
    if nb > 1 and value_scales.stride(0) != stride:
        raise _err(f"key/value scale strides differ: {stride} vs {value_scales.stride(0)}")
    return geometry + (stride,)


def reshape_and_cache_block_scaled(key: torch.Tensor, value: torch.Tensor,
                                   key_scales: torch.Tensor, value_scales: torch.Tensor,
                                   key_cache: torch.Tensor, value_cache: torch.Tensor,
                                   slot_mapping: torch.Tensor) -> None:
    """Scatter ``key``/``value`` [T, KVH, D] into the block-scaled caches at
    ``slot_mapping`` (i64), in place; negative slots are padding.

    ``key_scales``/``value_scales`` f32 [num_blocks, KVH] become, per block and head, the
    smallest power of two that brings the block's largest element into E4M3's range. A
    token at offset 0 of a block opens it (what it held no longer counts); a larger
    element later rescales the bytes that are there. Tokens of one block are neighbours
    in the call."""
    _same_device(key_cache, key, value, value_cache, slot_mapping, key_scales, value_scales)
    nb, kvh, d, bs, bstride, hstride, sstride = _geometry(key_cache, value_cache, key_scales,
                                                          value_scales)
    shape = key.shape
    if len(shape) != 3 or value.shape != shape:
        raise _err(f"key/value must be [T, KVH, D] of equal shape, got {tuple(key.shape)} and "
                   f"{tuple(value.shape)}")
    t, kh, kd = shape
    if kh != kvh or kd != d:
        raise _err(f"key shape {tuple(key.shape)} does not match cache heads={kvh} dim={d}")
    if key.dtype is not value.dtype:
        raise _err(f"key/value dtype mismatch: {key.dtype} vs {value.dtype}")
    if slot_mapping.dtype is not torch.int64 or slot_mapping.shape != (t,):
        raise _err(f"slot_mapping must be i64 [{t}], got {slot_mapping.dtype} "
                   f"{tuple(slot_mapping.shape)}")
    ks, kh, kd = key.stride()
    if kd != 1 or kh != d:
        key, ks = key.contiguous(), kvh * d
    vs, kh, kd = value.stride()
    if kd != 1 or kh != d:
        value, vs = value.contiguous(), kvh * d
    if t <= 1:  # (one token: its stride is free)
        ks = vs = kvh * d
    slot_mapping = slot_mapping.contiguous()
    with _on_device_of(key_cache):
        check(_lib.load().vpa_reshape_and_cache_block_scaled(
            key.data_ptr(), value.data_ptr(), ks, vs, key_scales.data_ptr(),
            value_scales.data_ptr(), sstride, key_cache.data_ptr(), value_cache.data_ptr(),
            slot_mapping.data_ptr(), t, kvh, d, bs, nb, bstride, hstride, dtype_code(key.dtype),
            _stream(key_cache)))


def paged_attention_block_scaled_workspace(num_seqs: int, num_heads: int, num_kv_heads: int,
                                           head_dim: int, max_context_len: int,
                                           dtype: torch.dtype, device, *, max_query_len: int = 1,
                                           total_query_rows: Optional[int] = None
                                           ) -> Optional[torch.Tensor]:
    """Caller-side workspace of ``paged_attention_block_scaled`` (None when not needed)."""
    rows = num_seqs * max_query_len if total_query_rows is None else total_query_rows
    n = _lib.load().vpa_paged_attention_block_scaled_workspace_size(
        num_seqs, max_query_len, max_context_len, rows, num_heads, num_kv_heads, head_dim,
        dtype_code(dtype))
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def paged_attention_block_scaled(q: torch.Tensor, key_scales: torch.Tensor,
                                 value_scales: torch.Tensor, key_cache: torch.Tensor,
                                 value_cache: torch.Tensor, block_tables: torch.Tensor,
                                 context_lens: torch.Tensor, softmax_scale: float, *,
                                 cu_seqlens_q: Optional[torch.Tensor] = None, causal: bool = True,
                                 max_query_len: Optional[int] = None,
                                 max_context_len: Optional[int] = None,
                                 denom_eps: Optional[float] = None,
                                 out: Optional[torch.Tensor] = None,
                                 workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of ``q`` [total_q, H, D] (bf16/f16/f32) over a block-scaled cache; returns
    the same shape.

    Without ``cu_seqlens_q`` row s is sequence s's one query (a decode step); with it
    (u32 [B + 1]) sequence s owns rows cu_seqlens_q[s] .. cu_seqlens_q[s + 1] - 1, the last
    tokens of its context_lens[s], and ``causal`` hides the tokens behind each row's own.
    The maxima size the grid; a caller that knows them on the host passes them to skip a
    device read. ``denom_eps`` is added to the softmax denominator: by default as
    ``paged_attention`` (1e-6) and ``paged_attention_varlen_prefill`` (0 where causal) do."""
    _same_device(q, key_cache, value_cache, key_scales, value_scales, block_tables, context_lens,
                 cu_seqlens_q, out, workspace)
    nb, kvh, d, bs, bstride, hstride, sstride = _geometry(key_cache, value_cache, key_scales,
                                                          value_scales)
    shape, tables = q.shape, block_tables.shape
    if len(shape) != 3 or shape[2] != d:
        raise _err(f"q must be [total_q, H, {d}], got {tuple(q.shape)}")
    rows, h, _ = shape
    if block_tables.dtype is not torch.uint32 or len(tables) != 2:
        raise _err(f"block_tables must be u32 2-d, got {block_tables.dtype} "
                   f"{tuple(block_tables.shape)}")
    b, cols = tables
    if context_lens.dtype is not torch.uint32 or context_lens.shape != (b,):
        raise _err(f"context_lens must be u32 [{b}], got {context_lens.dtype} "
                   f"{tuple(context_lens.shape)}")
    if cu_seqlens_q is None:
        if rows != b:
            raise _err(f"q has {rows} rows for {b} sequences: cu_seqlens_q is needed")
        max_query_len = 1
    elif cu_seqlens_q.dtype != torch.uint32 or cu_seqlens_q.shape != (b + 1,):
        raise _err(f"cu_seqlens_q must be u32 [{b + 1}], got {cu_seqlens_q.dtype} "
                   f"{tuple(cu_seqlens_q.shape)}")
    elif max_query_len is None:
        max_query_len = int((cu_seqlens_q[1:].long() - cu_seqlens_q[:-1].long()).max().item()) \
            if b else 0
    if max_context_len is None:
        max_context_len = int(context_lens.long().max().item()) if b else 0
    if denom_eps is None:
        denom_eps = 0.0 if causal and cu_seqlens_q is not None else 1e-6
    q = q.contiguous()
    block_tables = block_tables.contiguous()
    context_lens = context_lens.contiguous()
    if cu_seqlens_q is not None:
        cu_seqlens_q = cu_seqlens_q.contiguous()
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise _err("out must be a contiguous tensor shaped and typed like q")
    code = dtype_code(q.dtype)
    with _on_device_of(q):
        lib = _lib.load()
        if workspace is None:
            nbytes = lib.vpa_paged_attention_block_scaled_workspace_size(
                b, int(max_query_len), int(max_context_len), rows, h, kvh, d, code)
            if nbytes:
                workspace = context_lens.new_empty(((nbytes + 3) // 4,))
        else:
            nbytes = workspace.nbytes
        check(lib.vpa_paged_attention_block_scaled(
            out.data_ptr(), q.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(), sstride,
            key_cache.data_ptr(), value_cache.data_ptr(), block_tables.data_ptr(),
            cols, _ptr(cu_seqlens_q), context_lens.data_ptr(), b,
            int(max_query_len), int(max_context_len), rows, float(softmax_scale),
            float(denom_eps), int(bool(causal)), h, kvh, d, bs, nb, bstride, hstride, code,
            _ptr(workspace), nbytes, _stream(q)))
    return out
