"""Copies of cache blocks within their pools (``vpa_copy_blocks``), as forked and moved
blocks need them."""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import check
from .ops import _err, _on_device_of, _ptr, _require_device, _stream


def copy_blocks(buffers: Sequence[torch.Tensor], src_blocks: torch.Tensor,
                dst_blocks: torch.Tensor, num_pairs: Optional[torch.Tensor] = None) -> None:
    """Copies block src_blocks[p] to block dst_blocks[p] (u32 [P]) in each of ``buffers``,
    tensors whose first dimension counts the pool's blocks (K, V and scales of every
    layer) and whose blocks are contiguous. ``num_pairs`` (u32 [1], on the device) tells
    how many of the pairs there are. The destinations are distinct and none of them is a
    source; ids past the pool copy nothing."""
    _require_device(src_blocks, dst_blocks, num_pairs, *buffers)
    if src_blocks.dtype != torch.uint32 or src_blocks.dim() != 1 or \
            dst_blocks.dtype != torch.uint32 or dst_blocks.shape != src_blocks.shape:
        raise _err(f"src_blocks and dst_blocks must be u32 1-d of equal length, got "
                   f"{src_blocks.dtype} {tuple(src_blocks.shape)} and {dst_blocks.dtype} "
                   f"{tuple(dst_blocks.shape)}")
    if num_pairs is not None and (num_pairs.dtype != torch.uint32 or num_pairs.numel() != 1):
        raise _err(f"num_pairs must be u32 [1], got {num_pairs.dtype} {tuple(num_pairs.shape)}")
    n = len(buffers)
    if n == 0 or src_blocks.numel() == 0:
        return
    blocks = buffers[0].shape[0] if buffers[0].dim() else -1
    base, stride, size = (ctypes.c_void_p * n)(), (ctypes.c_int64 * n)(), (ctypes.c_int64 * n)()
    for k, t in enumerate(buffers):
        if t.dim() < 1 or t.shape[0] != blocks or not (blocks == 0 or t[0].is_contiguous()):
            raise _err(f"buffer {k} must be [{blocks}, ...] with contiguous blocks, got "
                       f"{tuple(t.shape)} of strides {t.stride()}")
        base[k], e = t.data_ptr(), t.element_size()
        size[k] = t.numel() // max(blocks, 1) * e
        stride[k] = t.stride(0) * e if blocks > 1 else size[k]
    if blocks == 0 or all(b == 0 for b in size):
        return
    src_blocks, dst_blocks = src_blocks.contiguous(), dst_blocks.contiguous()
    with _on_device_of(src_blocks):
        check(_lib.load().vpa_copy_blocks(
            base, stride, size, n, src_blocks.data_ptr(), dst_blocks.data_ptr(), _ptr(num_pairs),
            src_blocks.numel(), blocks, _stream(src_blocks)))
