"""Copies of cache blocks within their pools (``vpa_copy_blocks``), as forked and moved
blocks need them."""

from __future__ import annotations

from typing import Optional

import torch

from .ops import BlockBuffers, Buffers, _err, _on_device_of, _require_device


def copy_blocks(buffers: Buffers, src_blocks: torch.Tensor,
                dst_blocks: torch.Tensor, num_pairs: Optional[torch.Tensor] = None) -> None:
    """Copies block src_blocks[p] to block dst_blocks[p] (u32 [P]) in each of ``buffers``,
    tensors whose first dimension counts the pool's blocks (K, V and scales of every
    layer) and whose blocks are contiguous, or ``BlockBuffers`` of them. ``num_pairs``
    (u32 [1], on the device) tells how many of the pairs there are. The destinations are
    distinct and none of them is a source; ids past the pool copy nothing."""
    _require_device(src_blocks, dst_blocks, num_pairs)
    if src_blocks.dtype != torch.uint32 or src_blocks.dim() != 1 or \
            dst_blocks.dtype != torch.uint32 or dst_blocks.shape != src_blocks.shape:
        raise _err(f"src_blocks and dst_blocks must be u32 1-d of equal length, got "
                   f"{src_blocks.dtype} {tuple(src_blocks.shape)} and {dst_blocks.dtype} "
                   f"{tuple(dst_blocks.shape)}")
    if num_pairs is not None and (num_pairs.dtype != torch.uint32 or num_pairs.numel() != 1):
        raise _err(f"num_pairs must be u32 [1], got {num_pairs.dtype} {tuple(num_pairs.shape)}")
    pools = BlockBuffers.of(buffers, None, src_blocks.get_device())
    if src_blocks.numel() == 0:
        return
    src_blocks, dst_blocks = src_blocks.contiguous(), dst_blocks.contiguous()
    with _on_device_of(src_blocks):
        pools.copy(src_blocks, dst_blocks, num_pairs)
