"""Copies of cache blocks within their pools (``vpa_copy_blocks``), as forked and moved
blocks need them."""

from __future__ import annotations

from array import array
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import check
from .ops import _err, _on_device_of, _ptr, _require_device, _stream


class _Pools:
    """Addresses, strides and sizes of the blocks of ``buffers``, checked, in the host
    arrays that ``vpa_copy_blocks`` reads."""

    def __init__(self, buffers: Sequence[torch.Tensor], blocks: int, device: int):
        # (a hundred or more tensors per call: few calls for each)
        base, size, stride = [], [], []
        for t in buffers:
            if t.get_device() != device:
                _require_device(t)
                raise _err(f"device mismatch: a buffer on {t.device}, ids on cuda:{device}")
            if t.dim() < 1 or t.shape[0] != blocks:
                raise _err(f"buffers must be pools of {blocks} blocks, got {tuple(t.shape)}")
            if blocks and t.is_contiguous():
                n = t.nbytes // blocks
                stride.append(n)
            elif blocks:
                if not t[0].is_contiguous():
                    raise _err(f"buffers must have contiguous blocks, got {tuple(t.shape)} of "
                               f"strides {t.stride()}")
                n = t.numel() // blocks * t.element_size()
                stride.append(t.stride(0) * t.element_size() if blocks > 1 else n)
            if blocks and n:
                base.append(t.data_ptr())
                size.append(n)
            elif blocks:
                stride.pop()
        self.blocks, self.count = blocks, len(base)
        self.base, self.stride, self.size = array("Q", base), array("q", stride), array("q", size)

    def copy(self, src_blocks: torch.Tensor, dst_blocks: torch.Tensor,
             num_pairs: Optional[torch.Tensor]) -> None:
        """The copies of contiguous u32 pairs, on the current device and stream."""
        if self.count == 0:
            return
        check(_lib.load().vpa_copy_blocks(
            self.base.buffer_info()[0], self.stride.buffer_info()[0], self.size.buffer_info()[0],
            self.count, src_blocks.data_ptr(), dst_blocks.data_ptr(), _ptr(num_pairs),
            src_blocks.numel(), self.blocks, _stream(src_blocks)))


def copy_blocks(buffers: Sequence[torch.Tensor], src_blocks: torch.Tensor,
                dst_blocks: torch.Tensor, num_pairs: Optional[torch.Tensor] = None) -> None:
    """Copies block src_blocks[p] to block dst_blocks[p] (u32 [P]) in each of ``buffers``,
    tensors whose first dimension counts the pool's blocks (K, V and scales of every
    layer) and whose blocks are contiguous. ``num_pairs`` (u32 [1], on the device) tells
    how many of the pairs there are. The destinations are distinct and none of them is a
    source; ids past the pool copy nothing."""
    _require_device(src_blocks, dst_blocks, num_pairs)
    if src_blocks.dtype != torch.uint32 or src_blocks.dim() != 1 or \
            dst_blocks.dtype != torch.uint32 or dst_blocks.shape != src_blocks.shape:
        raise _err(f"src_blocks and dst_blocks must be u32 1-d of equal length, got "
                   f"{src_blocks.dtype} {tuple(src_blocks.shape)} and {dst_blocks.dtype} "
                   f"{tuple(dst_blocks.shape)}")
    if num_pairs is not None and (num_pairs.dtype != torch.uint32 or num_pairs.numel() != 1):
        raise _err(f"num_pairs must be u32 [1], got {num_pairs.dtype} {tuple(num_pairs.shape)}")
    if len(buffers) == 0:
        return
    blocks = buffers[0].shape[0] if buffers[0].dim() else 0
    pools = _Pools(buffers, blocks, src_blocks.get_device())
    if src_blocks.numel() == 0:
        return
    src_blocks, dst_blocks = src_blocks.contiguous(), dst_blocks.contiguous()
    with _on_device_of(src_blocks):
        pools.copy(src_blocks, dst_blocks, num_pairs)
