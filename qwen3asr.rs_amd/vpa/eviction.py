"""Eviction of cached tokens by accumulated attention weight: the weights each
cached token gets (``vpa_paged_attention_weights``) and the cut of a cache to a
budget of tokens by them (``vpa_evict_kv_cache``)."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import check
from .ops import _err, _on_device_of, _ptr, _require_device, _stream, cache_geometry, dtype_code


def _check_tables(block_tables: torch.Tensor, context_lens: torch.Tensor) -> int:
    if block_tables.dtype != torch.uint32 or block_tables.dim() != 2:
        raise _err(f"block_tables must be u32 2-d, got {block_tables.dtype} "
                   f"{tuple(block_tables.shape)}")
    b = block_tables.shape[0]
    if context_lens.dtype != torch.uint32 or context_lens.shape != (b,):
        raise _err(f"context_lens must be u32 [{b}], got {context_lens.dtype} "
                   f"{tuple(context_lens.shape)}")
    return b


def _score_strides(scores: torch.Tensor, b: int, kvh: int, max_context_len: int):
    if scores.dtype != torch.float32 or scores.dim() != 3 or scores.shape[:2] != (b, kvh) or \
            scores.shape[2] < max_context_len:
        raise _err(f"scores must be f32 [{b}, {kvh}, >= {max_context_len}], got {scores.dtype} "
                   f"{tuple(scores.shape)}")
    if scores.stride(2) != 1 and scores.shape[2] > 1:
        raise _err("scores must be contiguous along the tokens")
    width = scores.shape[2]
    head = scores.stride(1) if kvh > 1 else width
    return scores.stride(0) if b > 1 else head * kvh, head


def paged_attention_weights_workspace(total_query_rows: int, num_heads: int,
                                      max_context_len: int, device, *,
                                      max_query_len: Optional[int] = None,
                                      num_kv_heads: Optional[int] = None
                                      ) -> Optional[torch.Tensor]:
    """Caller-side workspace of ``paged_attention_weights`` (None when not needed). With
    ``max_query_len`` and ``num_kv_heads`` that of calls of these sizes: where a kv head
    can have more than 16 rows in a sequence (a prompt's) 8 bytes per row, head and 256
    tokens in place of 1032."""
    lib = _lib.load()
    if max_query_len is None or num_kv_heads is None:
        n = lib.vpa_paged_attention_weights_workspace_size(total_query_rows, num_heads,
                                                           max_context_len)
    else:
        n = lib.vpa_paged_attention_weights_call_workspace_size(
            total_query_rows, max_query_len, max_context_len, num_heads, num_kv_heads)
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def paged_attention_weights(q: torch.Tensor, key_cache: torch.Tensor,
                            k_scale: Optional[torch.Tensor], block_tables: torch.Tensor,
                            context_lens: torch.Tensor, softmax_scale: float,
                            scores: torch.Tensor, *, cu_seqlens_q: Optional[torch.Tensor] = None,
                            causal: bool = True, max_query_len: Optional[int] = None,
                            max_context_len: Optional[int] = None,
                            workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Adds to ``scores`` (f32 [B, KVH, width], width >= max_context_len, updated in
    place and returned) the softmax weight each cached token gets from the query
    rows ``q`` [rows, H, D], summed over the rows of its sequence and the query
    heads of its kv head.

    Without ``cu_seqlens_q`` row s belongs to sequence s (a decode step);
    with it (u32 [B + 1]) a sequence has several rows, its last tokens, and
    with ``causal`` each sees the tokens up to its own. ``max_query_len`` and
    ``max_context_len`` size the launch; a caller that knows them on the host
    passes them to skip a device read.

    A sequence of length 0 adds nothing. A row that did not run in a step
    (``DeviceBlockAllocator.step``: negative slot) has context_lens 1, which would add
    a whole weight to its first token; give it 0:
    ``(context_lens.view(torch.int32) * (slot_mapping >= 0)).view(torch.uint32)``."""
    _require_device(q, key_cache, k_scale, block_tables, context_lens, scores, cu_seqlens_q,
                    workspace)
    if key_cache.dim() != 5:
        raise _err(f"key_cache must be 5-d, got {tuple(key_cache.shape)}")
    nb, kvh, dx, bs, x = key_cache.shape
    d = dx * x
    if x * key_cache.element_size() != 16 or key_cache.stride()[2:] != (bs * x, x, 1):
        raise _err("paged cache tiles must be contiguous, 16-byte packs")
    if q.dim() != 3 or q.shape[2] != d:
        raise _err(f"q must be [rows, H, {d}], got {tuple(q.shape)}")
    rows, h, _ = q.shape
    b = _check_tables(block_tables, context_lens)
    if cu_seqlens_q is None:
        if rows != b:
            raise _err(f"q must have a row per sequence ({b}) without cu_seqlens_q, got {rows}")
        max_query_len = 1
    elif cu_seqlens_q.dtype != torch.uint32 or cu_seqlens_q.shape != (b + 1,):
        raise _err(f"cu_seqlens_q must be u32 [{b + 1}], got {cu_seqlens_q.dtype} "
                   f"{tuple(cu_seqlens_q.shape)}")
    elif max_query_len is None:
        max_query_len = int((cu_seqlens_q[1:].long() - cu_seqlens_q[:-1].long()).max().item()) \
            if b else 0
    if max_context_len is None:
        max_context_len = int(context_lens.long().max().item()) if b else 0
    seq_stride, head_stride = _score_strides(scores, b, kvh, int(max_context_len))
    q = q.contiguous()
    block_tables = block_tables.contiguous()
    context_lens = context_lens.contiguous()
    if cu_seqlens_q is not None:
        cu_seqlens_q = cu_seqlens_q.contiguous()
    with _on_device_of(q):
        lib = _lib.load()
        if workspace is None:
            nbytes = lib.vpa_paged_attention_weights_call_workspace_size(
                rows, int(max_query_len), int(max_context_len), h, kvh)
            workspace = context_lens.new_empty(((nbytes + 3) // 4,))
        else:
            nbytes = workspace.nbytes
        check(lib.vpa_paged_attention_weights(
            scores.data_ptr(), seq_stride, head_stride, q.data_ptr(), _ptr(k_scale),
            key_cache.data_ptr(), block_tables.data_ptr(), block_tables.shape[1],
            _ptr(cu_seqlens_q), context_lens.data_ptr(), b, int(max_query_len),
            int(max_context_len), rows, float(softmax_scale), int(causal), h, kvh, d, bs, nb,
            key_cache.stride(0), key_cache.stride(1), dtype_code(q.dtype),
            dtype_code(key_cache.dtype), workspace.data_ptr(), nbytes, _stream(q)))
    return scores


def evict_kv_cache_workspace(num_seqs: int, num_kv_heads: int, max_context_len: int,
                             block_size: int, device) -> Optional[torch.Tensor]:
    """Caller-side workspace of ``evict_kv_cache`` (None when not needed)."""
    n = _lib.load().vpa_evict_kv_cache_workspace_size(num_seqs, num_kv_heads, max_context_len,
                                                      block_size)
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def evict_kv_cache(key_cache: torch.Tensor, value_cache: torch.Tensor, scores: torch.Tensor,
                   block_tables: torch.Tensor, context_lens: torch.Tensor, budget: int, *,
                   keep_first: int = 0, keep_last: int = 0,
                   max_context_len: Optional[int] = None,
                   new_context_lens: Optional[torch.Tensor] = None,
                   kept: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cuts each sequence of more than ``budget`` tokens to ``budget`` per kv head:
    its first ``keep_first``, its last ``keep_last`` and the others with the
    highest ``scores`` [B, KVH, width] (equal ones: the earlier) stay, moved to the
    front in their order in the caches and the scores (in place).

    Returns (new_context_lens u32 [B], kept u32 [B, KVH, budget]: the old
    position of each token that stayed, 0xffffffff past the last). The blocks past
    ceil(new_context_lens / block_size) may then be given back
    (``DeviceBlockAllocator.trim``, with the step's slot_mapping where rows may not
    have run: their new length is not what they hold)."""
    _require_device(key_cache, value_cache, scores, block_tables, context_lens, new_context_lens,
                    kept, workspace)
    nb, kvh, d, bs, bstride, hstride = cache_geometry(key_cache, value_cache)
    b = _check_tables(block_tables, context_lens)
    if max_context_len is None:
        max_context_len = int(context_lens.long().max().item()) if b else 0
    seq_stride, head_stride = _score_strides(scores, b, kvh, int(max_context_len))
    if new_context_lens is None:
        new_context_lens = context_lens.new_empty((b,))
    elif new_context_lens.dtype != torch.uint32 or new_context_lens.shape != (b,) or \
            not new_context_lens.is_contiguous():
        raise _err(f"new_context_lens must be a contiguous u32 [{b}] tensor")
    if kept is None:
        kept = context_lens.new_empty((b, kvh, max(int(budget), 0)))
    elif kept.dtype != torch.uint32 or kept.shape != (b, kvh, budget) or not kept.is_contiguous():
        raise _err(f"kept must be a contiguous u32 [{b}, {kvh}, {budget}] tensor")
    block_tables = block_tables.contiguous()
    context_lens = context_lens.contiguous()
    with _on_device_of(scores):
        lib = _lib.load()
        if workspace is None:
            nbytes = lib.vpa_evict_kv_cache_workspace_size(b, kvh, int(max_context_len), bs)
            workspace = context_lens.new_empty(((nbytes + 3) // 4,))
        else:
            nbytes = workspace.nbytes
        check(lib.vpa_evict_kv_cache(
            key_cache.data_ptr(), value_cache.data_ptr(), scores.data_ptr(), seq_stride,
            head_stride, block_tables.data_ptr(), block_tables.shape[1], context_lens.data_ptr(),
            new_context_lens.data_ptr(), kept.data_ptr(), b, int(max_context_len), int(budget),
            int(keep_first), int(keep_last), kvh, d, bs, nb, bstride, hstride,
            dtype_code(key_cache.dtype), workspace.data_ptr(), nbytes, _stream(scores)))
    return new_context_lens, kept
