"""Verification of drafted tokens against the target's logits
(``vpa_verify_draft_tokens``), the sampling counterpart of
``argmax_token_ids_from_logits``."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import check
from .ops import _err, _on_device_of, _ptr, _require_device, _stream, dtype_code


def verify_draft_tokens_workspace(num_seqs: int, max_drafts: int, vocab: int,
                                  device) -> Optional[torch.Tensor]:
    """Caller-side workspace of ``verify_draft_tokens`` (None when not needed)."""
    n = _lib.load().vpa_verify_draft_tokens_workspace_size(num_seqs, max_drafts, vocab)
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _device_vector(name: str, t: Optional[torch.Tensor], dtype, shape) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype != dtype or t.shape != shape:
        raise _err(f"{name} must be {dtype} {list(shape)}, got {t.dtype} {tuple(t.shape)}")
    return t.contiguous()


def verify_draft_tokens(target_logits: torch.Tensor, draft_ids: torch.Tensor,
                        accept_u: torch.Tensor, sample_u: torch.Tensor, *,
                        draft_logits: Optional[torch.Tensor] = None,
                        num_drafts: Optional[torch.Tensor] = None,
                        temperature: Optional[torch.Tensor] = None,
                        out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                        workspace: Optional[torch.Tensor] = None
                        ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Accepts or replaces the drafts of each sequence so that the emitted tokens are
    distributed as the target's own; returns (ids u32 [B, K + 1], count u32 [B]):
    the first count[b] ids of a row are emitted, 0xffffffff follows.

    ``target_logits`` [B, K + 1, V] (row i follows draft i - 1), ``draft_ids`` u32
    [B, K], ``accept_u`` f32 [B, K] and ``sample_u`` f32 [B] uniform in [0, 1),
    ``draft_logits`` [B, K, V] the drafts were drawn from (None: looked up,
    probability 1), ``num_drafts`` u32 [B] (None: K each), ``temperature`` f32 [B]
    (None: 1; <= 0: greedy). K = 0 samples one token per sequence."""
    _require_device(target_logits, draft_ids, accept_u, sample_u, draft_logits, num_drafts,
                    temperature, workspace, *(out or ()))
    if target_logits.dim() != 3 or target_logits.shape[1] < 1:
        raise _err(f"target_logits must be [B, K + 1, V], got {tuple(target_logits.shape)}")
    b, k1, v = target_logits.shape
    k = k1 - 1
    draft_ids = _device_vector("draft_ids", draft_ids, torch.uint32, (b, k))
    accept_u = _device_vector("accept_u", accept_u, torch.float32, (b, k))
    sample_u = _device_vector("sample_u", sample_u, torch.float32, (b,))
    num_drafts = _device_vector("num_drafts", num_drafts, torch.uint32, (b,))
    temperature = _device_vector("temperature", temperature, torch.float32, (b,))
    if target_logits.stride(2) != 1 and v > 1:
        target_logits = target_logits.contiguous()
    ds = dr = 0
    if draft_logits is not None:
        if draft_logits.dtype != target_logits.dtype or draft_logits.shape != (b, k, v):
            raise _err(f"draft_logits must be {target_logits.dtype} [{b}, {k}, {v}], got "
                       f"{draft_logits.dtype} {tuple(draft_logits.shape)}")
        if draft_logits.stride(2) != 1 and v > 1:
            draft_logits = draft_logits.contiguous()
        ds, dr = draft_logits.stride(0), draft_logits.stride(1)
    if out is None:
        ids, count = draft_ids.new_empty((b, k1)), draft_ids.new_empty((b,))
    else:
        ids, count = out
        if ids.dtype != torch.uint32 or ids.shape != (b, k1) or not ids.is_contiguous() or \
                count.dtype != torch.uint32 or count.shape != (b,) or not count.is_contiguous():
            raise _err(f"out must be contiguous u32 [{b}, {k1}] and [{b}] tensors")
    with _on_device_of(target_logits):
        lib = _lib.load()
        if workspace is None:
            nbytes = lib.vpa_verify_draft_tokens_workspace_size(b, k, v)
            workspace = draft_ids.new_empty(((nbytes + 3) // 4,))
        else:
            nbytes = workspace.nbytes
        check(lib.vpa_verify_draft_tokens(
            ids.data_ptr(), count.data_ptr(), target_logits.data_ptr(), target_logits.stride(0),
            target_logits.stride(1), _ptr(draft_logits), ds, dr, draft_ids.data_ptr(),
            _ptr(num_drafts), _ptr(temperature), accept_u.data_ptr(), sample_u.data_ptr(), b, k, v,
            dtype_code(target_logits.dtype), workspace.data_ptr(), nbytes, _stream(target_logits)))
    return ids, count
