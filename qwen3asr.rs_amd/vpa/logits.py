"""Penalties for repeated tokens, biases and grammar masks on logits
(``vpa_adjust_logits``), before a token is chosen by ``argmax_token_ids_from_logits`` or
``verify_draft_tokens``."""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._lib import check
from .ops import _err, _on_device_of, _ptr, _same_device, _stream, dtype_code


def _list(name: str, ids: Optional[torch.Tensor], lengths: Optional[torch.Tensor], b: int):
    """A list of ids per sequence and its lengths, as the entry point takes them."""
    if ids is None:
        if lengths is not None:
            raise _err(f"the lengths of {name} come without {name}")
        return None, 0, None
    if ids.dtype != torch.uint32 or ids.dim() != 2 or ids.shape[0] != b:
        raise _err(f"{name} must be u32 [{b}, entries], got {ids.dtype} {tuple(ids.shape)}")
    if lengths is not None:
        if lengths.dtype != torch.uint32 or lengths.shape != (b,):
            raise _err(f"the lengths of {name} must be u32 [{b}], got {lengths.dtype} "
                       f"{tuple(lengths.shape)}")
        lengths = lengths.contiguous()
    return ids.contiguous(), ids.shape[1], lengths


def _per_sequence(name: str, t: Optional[torch.Tensor], b: int) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype != torch.float32 or t.shape != (b,):
        raise _err(f"{name} must be f32 [{b}], got {t.dtype} {tuple(t.shape)}")
    return t.contiguous()


def adjust_logits(logits: torch.Tensor, generated: Optional[torch.Tensor] = None,
                  gen_len: Optional[torch.Tensor] = None, *,
                  prompt: Optional[torch.Tensor] = None,
                  prompt_len: Optional[torch.Tensor] = None,
                  draft_ids: Optional[torch.Tensor] = None,
                  repetition: Optional[torch.Tensor] = None,
                  presence: Optional[torch.Tensor] = None,
                  frequency: Optional[torch.Tensor] = None,
                  bias_ids: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                  bias_len: Optional[torch.Tensor] = None,
                  allowed: Optional[torch.Tensor] = None,
                  allowed_rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Adjusts ``logits`` [B, V], or [B, K + 1, V] for K drafted tokens, in place and returns
    them.

    With c the occurrences of a token in ``generated`` [B, capacity] u32 (its first
    gen_len[b]) and, for row i, in draft_ids[b, :i] (u32 [B, K]): where c > 0 or the token
    is in ``prompt`` (u32 [B, P], prompt_len u32 [B]) a positive logit is divided by
    ``repetition``[b] and any other multiplied; then frequency[b] * c and, where c > 0,
    presence[b] are subtracted (f32 [B] each, None: none). ``bias`` f32 [B, N] is added to
    the tokens bias_ids u32 [B, N] (the first bias_len[b]; of equal ids the last counts).
    ``allowed`` u32 [M, >= ceil(V / 32)] are masks of one bit per token: a row takes mask
    allowed_rows[b] or allowed_rows[b, i] (u32; one >= M: none; None: the mask of its
    index) and what its mask leaves out becomes -inf."""
    _same_device(logits, generated, gen_len, prompt, prompt_len, draft_ids, repetition, presence,
                 frequency, bias_ids, bias, bias_len, allowed, allowed_rows)
    shape, strides = logits.shape, logits.stride()
    if len(shape) == 3:
        b, k1, v = shape
    elif len(shape) == 2:
        (b, v), k1 = shape, 1
    else:
        raise _err(f"logits must be [B, V] or [B, K + 1, V], got {tuple(logits.shape)}")
    if v > 1 and strides[-1] != 1:
        raise _err("logits must be contiguous along the vocabulary")
    gen, gen_cap, gen_len = _list("generated", generated, gen_len, b)
    pro, pro_cap, prompt_len = _list("prompt", prompt, prompt_len, b)
    ids, bias_cap, bias_len = _list("bias_ids", bias_ids, bias_len, b)
    repetition = _per_sequence("repetition", repetition, b)
    presence = _per_sequence("presence", presence, b)
    frequency = _per_sequence("frequency", frequency, b)
    if draft_ids is not None:
        if draft_ids.dtype != torch.uint32 or draft_ids.shape != (b, k1 - 1):
            raise _err(f"draft_ids must be u32 [{b}, {k1 - 1}], got {draft_ids.dtype} "
                       f"{tuple(draft_ids.shape)}")
        draft_ids = draft_ids.contiguous() if k1 > 1 else None
    if (bias is None) != (ids is None) or (bias is not None and (
            bias.dtype != torch.float32 or bias.shape != ids.shape)):
        raise _err("bias must be f32 of the shape of bias_ids")
    bias = None if bias is None else bias.contiguous()
    masks = width = 0
    if allowed is not None:
        if allowed.dtype != torch.uint32 or allowed.dim() != 2:
            raise _err(f"allowed must be u32 [M, words], got {allowed.dtype} "
                       f"{tuple(allowed.shape)}")
        allowed = allowed.contiguous()
        masks, width = allowed.shape
    if allowed_rows is not None:
        if allowed is None:
            raise _err("allowed_rows comes without allowed")
        if allowed_rows.dtype != torch.uint32 or allowed_rows.numel() != b * k1 or \
                allowed_rows.shape[0] != b:
            raise _err(f"allowed_rows must be u32 of the {b} x {k1} rows, got "
                       f"{allowed_rows.dtype} {tuple(allowed_rows.shape)}")
        allowed_rows = allowed_rows.contiguous()
    # (a dimension of one row has a free stride)
    row = strides[1] if k1 > 1 else v
    seq = strides[0] if b > 1 else row * k1
    with _on_device_of(logits):
        check(_lib.load().vpa_adjust_logits(
            logits.data_ptr(), seq, row, b, k1, v, dtype_code(logits.dtype), _ptr(gen), gen_cap,
            _ptr(gen_len), _ptr(pro), pro_cap, _ptr(prompt_len), _ptr(draft_ids),
            _ptr(repetition), _ptr(presence), _ptr(frequency), _ptr(ids), _ptr(bias), bias_cap,
            _ptr(bias_len), _ptr(allowed), masks, width, _ptr(allowed_rows), _stream(logits)))
    return logits
