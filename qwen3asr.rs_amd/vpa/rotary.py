"""Rotary positions of several axes on new q and k rows, alone or together
with the append to the paged cache (``vpa_rotary_qk``,
``vpa_rotary_reshape_and_cache``): the step between the projections and
``reshape_and_cache`` of a decoder layer
(``vasr-models/src/model/thinker_text.rs:1041-1068``)."""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from ._lib import check
from .ops import _err, _on_device_of, _ptr, _require_device, _stream, cache_geometry, dtype_code


def rotary_frequencies(rotary_dim: int, theta: float, device, *,
                       sections: Optional[Sequence[int]] = None, interleaved: bool = False
                       ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(inv_freq f64 [rotary_dim / 2], axes u8 [rotary_dim / 2]) for the rotary ops:
    inv_freq[i] = theta ** (-2 i / rotary_dim), and the position axis of each pair.

    ``sections`` gives the pairs of each axis (time, height, width, ...),
    summing to rotary_dim / 2; None: one axis. They lie one after the other,
    or with ``interleaved`` in turn (pair i belongs to axis a = i % len(sections)
    as long as that axis has pairs left, i < len(sections) * sections[a], and to
    axis 0 behind)."""
    half = rotary_dim // 2
    if rotary_dim < 2 or rotary_dim % 2:
        raise _err(f"rotary_dim must be even and positive, got {rotary_dim}")
    sec = [half] if sections is None else [int(n) for n in sections]
    if sum(sec) != half or min(sec) < 0:
        raise _err(f"sections {sec} must sum to rotary_dim / 2 = {half}")
    inv_freq = torch.tensor([float(theta) ** (-2.0 * i / rotary_dim) for i in range(half)],
                            dtype=torch.float64, device=device)
    axes = [a for a, n in enumerate(sec) for _ in range(n)]
    if interleaved:
        axes = [0] * half
        for i in range(half):
            a = i % len(sec)
            axes[i] = a if i < len(sec) * sec[a] else 0
    return inv_freq, torch.tensor(axes, dtype=torch.uint8, device=device)


def _rows(name: str, t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """([T, heads, D] with contiguous heads, as it is or copied; its token stride)."""
    if t.dim() != 3:
        raise _err(f"{name} must be [T, heads, D], got {tuple(t.shape)}")
    n, h, d = t.shape
    st, sh, sd = t.stride()
    if sd != 1 or (sh != d and h > 1) or (st < h * d and n > 1):
        return t.contiguous(), h * d
    # (a single row's stride is never stepped over: torch leaves anything there)
    return t, st if n > 1 else h * d


def _tables(positions, inv_freq, axes, tokens):
    """(position pointer, axis stride, int64?, num_axes, rotary_dim), checked."""
    if positions.dim() == 1:
        positions = positions[None]
    if positions.dim() != 2 or positions.shape[1] != tokens or \
            positions.dtype not in (torch.int64, torch.uint32):
        raise _err(f"positions must be i64 or u32 [axes, {tokens}], got {positions.dtype} "
                   f"{tuple(positions.shape)}")
    if positions.stride(1) != 1 and tokens > 1:
        positions = positions.contiguous()
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise _err(f"inv_freq must be contiguous f64 [rotary_dim / 2], got {inv_freq.dtype} "
                   f"{tuple(inv_freq.shape)}")
    if axes is not None and (axes.dtype != torch.uint8 or axes.shape != inv_freq.shape or
                             not axes.is_contiguous()):
        raise _err(f"axes must be contiguous u8 [{inv_freq.shape[0]}], got {axes.dtype} "
                   f"{tuple(axes.shape)}")
    n = positions.shape[0]
    stride = positions.stride(0) if n > 1 else 0
    return positions, stride, int(positions.dtype == torch.int64), n, 2 * inv_freq.shape[0]


def _norm(name: str, w: Optional[torch.Tensor], like: torch.Tensor) -> Optional[torch.Tensor]:
    if w is not None and (w.dtype != like.dtype or w.shape != like.shape[2:] or
                          not w.is_contiguous()):
        raise _err(f"{name} must be contiguous {like.dtype} [{like.shape[2]}], got {w.dtype} "
                   f"{tuple(w.shape)}")
    return w


def _out(name: str, out: Optional[torch.Tensor], like: torch.Tensor) -> Tuple[torch.Tensor, int]:
    if out is None:
        return (torch.empty_like(like, memory_format=torch.contiguous_format),
                like.shape[1] * like.shape[2])
    rows, stride = _rows(name, out)
    if out.shape != like.shape or out.dtype != like.dtype or rows is not out:
        raise _err(f"{name} must be shaped and typed like its input, heads contiguous")
    return out, stride


def rotary_qk(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
              axes: Optional[torch.Tensor] = None, *, q_norm: Optional[torch.Tensor] = None,
              k_norm: Optional[torch.Tensor] = None, norm_eps: float = 1e-6,
              adjacent: bool = False, out_q: Optional[torch.Tensor] = None,
              out_k: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``q`` [T, H, D] and ``k`` [T, KVH, D] (f32, f16 or bf16; slices of a packed
    projection are taken as they are) normalised per head row where ``q_norm`` /
    ``k_norm`` [D] are given and rotated; returns (q, k).

    ``positions`` [axes, T] (or [T]) i64 or u32; ``inv_freq`` and ``axes`` as
    ``rotary_frequencies`` gives them. Split pairs (i, i + R/2), or with
    ``adjacent`` (2i, 2i + 1). ``out_q`` / ``out_k`` may be q and k themselves."""
    _require_device(q, k, positions, inv_freq, axes, q_norm, k_norm, out_q, out_k)
    (q, qs), (k, ks) = _rows("q", q), _rows("k", k)
    t, h, d = q.shape
    if k.shape[0] != t or k.shape[2] != d or k.dtype != q.dtype:
        raise _err(f"k must be {q.dtype} [{t}, kv_heads, {d}], got {k.dtype} {tuple(k.shape)}")
    positions, stride, is64, num_axes, rot = _tables(positions, inv_freq, axes, t)
    _norm("q_norm", q_norm, q)
    _norm("k_norm", k_norm, k)
    (out_q, oqs), (out_k, oks) = _out("out_q", out_q, q), _out("out_k", out_k, k)
    with _on_device_of(q):
        check(_lib.load().vpa_rotary_qk(
            out_q.data_ptr(), out_k.data_ptr(), q.data_ptr(), k.data_ptr(), oqs, oks, qs, ks,
            positions.data_ptr(), stride, is64, inv_freq.data_ptr(), _ptr(axes), num_axes, rot,
            int(adjacent), _ptr(q_norm), _ptr(k_norm), float(norm_eps), t, h, k.shape[1], d,
            dtype_code(q.dtype), _stream(q)))
    return out_q, out_k


def rotary_reshape_and_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                             positions: torch.Tensor, inv_freq: torch.Tensor,
                             axes: Optional[torch.Tensor], k_scale: Optional[torch.Tensor],
                             v_scale: Optional[torch.Tensor], key_cache: torch.Tensor,
                             value_cache: torch.Tensor, slot_mapping: torch.Tensor, *,
                             q_norm: Optional[torch.Tensor] = None,
                             k_norm: Optional[torch.Tensor] = None, norm_eps: float = 1e-6,
                             adjacent: bool = False, out: Optional[torch.Tensor] = None
                             ) -> torch.Tensor:
    """``rotary_qk`` of ``q`` and ``k``, then ``reshape_and_cache`` of the rotated k
    and of ``v`` at ``slot_mapping``, in one launch; returns the rotated q. The
    caches are written in place, each key rounded once, to the cache's type."""
    _require_device(q, k, v, positions, inv_freq, axes, k_scale, v_scale, key_cache, value_cache,
                    slot_mapping, q_norm, k_norm, out)
    nb, kvh, d, bs, bstride, hstride = cache_geometry(key_cache, value_cache)
    (q, qs), (k, ks), (v, vs) = _rows("q", q), _rows("k", k), _rows("v", v)
    t, h, qd = q.shape
    if qd != d or k.shape != (t, kvh, d) or v.shape != k.shape:
        raise _err(f"q, k and v must be [{t}, heads, {d}] and twice [{t}, {kvh}, {d}], got "
                   f"{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise _err(f"q, k and v must be of one dtype, got {q.dtype}, {k.dtype} and {v.dtype}")
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (t,):
        raise _err(f"slot_mapping must be i64 [{t}], got {slot_mapping.dtype} "
                   f"{tuple(slot_mapping.shape)}")
    positions, stride, is64, num_axes, rot = _tables(positions, inv_freq, axes, t)
    _norm("q_norm", q_norm, q)
    _norm("k_norm", k_norm, k)
    out, outs = _out("out", out, q)
    slot_mapping = slot_mapping.contiguous()
    with _on_device_of(q):
        check(_lib.load().vpa_rotary_reshape_and_cache(
            out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), outs, qs, ks, vs,
            positions.data_ptr(), stride, is64, inv_freq.data_ptr(), _ptr(axes), num_axes, rot,
            int(adjacent), _ptr(q_norm), _ptr(k_norm), float(norm_eps), _ptr(k_scale),
            _ptr(v_scale), key_cache.data_ptr(), value_cache.data_ptr(), slot_mapping.data_ptr(), t, h, kvh, d, bs, nb, bstride, hstride,
            dtype_code(q.dtype), dtype_code(key_cache.dtype), _stream(q)))
    return out
