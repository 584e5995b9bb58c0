"""Refusals of the rotary, weights, eviction and verification entry points, on the
host before any launch (no GPU here), and their Python wrappers' checks."""

import ctypes

import pytest
import torch

import vpa
from vpa import _lib

INV, UNS, WS = (_lib.VPA_ERR_INVALID_ARGUMENT, _lib.VPA_ERR_UNSUPPORTED, _lib.VPA_ERR_WORKSPACE)
P = 1 << 20  # 256-byte aligned non-null host value standing in for a device pointer
BF16, F32, FP8 = _lib.DTYPE_BF16, _lib.DTYPE_F32, _lib.DTYPE_FP8_E4M3


def call(fn, base, over):
    args = dict(base)
    unknown = set(over) - set(args)
    assert not unknown, unknown
    args.update(over)
    lib = _lib.load()
    rc = getattr(lib, fn)(*args.values())
    return rc, lib.vpa_last_error().decode()


def refused(fn, base, over, code, needle):
    rc, msg = call(fn, base, over)
    assert rc == code and needle in msg, (rc, msg)


QK = dict(oq=P, ok=P, q=P, k=2 * P, oqs=2048, oks=1024, qs=2048, ks=1024, pos=P, ps=0, i64=1, freq=P,
          axes=P, n_axes=1, rot=128, adj=0, qn=None, kn=None, eps=1e-6, t=4, h=16, kvh=8, d=128,
          dtype=BF16, stream=None)


@pytest.mark.parametrize("over,code,needle", [
    (dict(dtype=FP8), UNS, "dtype"), (dict(dtype=9), UNS, "dtype"),
    (dict(t=-1), INV, "num_tokens"), (dict(h=0), INV, "num_heads"), (dict(kvh=0), INV, "num_kv_heads"),
    (dict(d=120), UNS, "head_dim"), (dict(d=272), UNS, "head_dim"), (dict(d=0), UNS, "head_dim"),
    (dict(rot=120), UNS, "rotary_dim"), (dict(rot=144), UNS, "rotary_dim"),
    (dict(rot=-16), UNS, "rotary_dim"), (dict(n_axes=0), UNS, "num_axes"),
    (dict(n_axes=5), UNS, "num_axes"), (dict(eps=-1.0), INV, "norm_eps"),
    (dict(eps=float("nan")), INV, "norm_eps"), (dict(eps=float("inf")), INV, "norm_eps"),
    (dict(ps=3), INV, "axis stride"), (dict(q=None), INV, "non-null"), (dict(k=None), INV, "non-null"),
    (dict(oq=None), INV, "non-null"), (dict(ok=None), INV, "out_key"), (dict(pos=None), INV, "non-null"),
    (dict(freq=None), INV, "non-null"), (dict(qs=2047), INV, "strides"), (dict(oks=1008), INV, "strides"),
    (dict(oq=P, q=P, oqs=4096), INV, "in place"), (dict(q=P + 2), INV, "aligned"),
    (dict(qn=P + 8), INV, "aligned"), (dict(ks=1028), INV, "aligned"), (dict(freq=P + 8), INV, "aligned"),
    (dict(axes=P + 1), INV, "aligned"), (dict(pos=P + 4), INV, "aligned"),
    (dict(t=1 << 24), INV, "too many tokens"),
])
def test_rotary_qk_rejects(over, code, needle):
    refused("vpa_rotary_qk", QK, over, code, needle)


def test_no_tokens_is_a_no_op():
    assert call("vpa_rotary_qk", QK, dict(t=0, q=None, k=None, oq=None, ok=None))[0] == 0
    assert call("vpa_rotary_reshape_and_cache", RC, dict(t=0, q=None, k=None, v=None, oq=None))[0] == 0


RC = dict(oq=P, q=P, k=2 * P, v=3 * P, oqs=2048, qs=2048, ks=1024, vs=1024, pos=P, ps=0, i64=1, freq=P,
          axes=None, n_axes=1, rot=128, adj=0, qn=None, kn=None, eps=1e-6, ksc=None, vsc=None, kc=P,
          vc=P, slots=P, t=4, h=16, kvh=8, d=128, bs=16, nb=10, bst=8 * 2048, hst=2048, dtype=BF16,
          cdtype=BF16, stream=None)


@pytest.mark.parametrize("over,code,needle", [
    (dict(cdtype=F32), UNS, "differs"), (dict(cdtype=FP8), INV, "k_scale"),
    (dict(cdtype=FP8, ksc=P, vsc=P + 2), INV, "aligned"), (dict(d=112, rot=112), UNS, "no kernel"),
    (dict(bs=24), UNS, "no kernel"), (dict(hst=100), INV, "strides"), (dict(kc=None), INV, "non-null"),
    (dict(h=12), INV, "multiple of"), (dict(v=None), INV, "value"), (dict(slots=None), INV, "slot_mapping"),
    (dict(vs=1000), INV, "value token stride"), (dict(v=P + 4), INV, "value rows"),
    (dict(rot=130), UNS, "rotary_dim"), (dict(nb=0), INV, "positive"), (dict(t=1 << 23), INV, "too many"),
])
def test_rotary_cache_rejects(over, code, needle):
    refused("vpa_rotary_reshape_and_cache", RC, over, code, needle)


def ws_bytes(rows, h, ctx):
    return _lib.load().vpa_paged_attention_weights_workspace_size(rows, h, ctx)


WT = dict(sc=P, ss=8 * 512, sh=512, q=P, ks=None, kc=P, bt=P, bts=32, cu=P, cl=P, n=4, mq=3, mc=500,
          rows=9, scale=0.1, causal=1, h=16, kvh=8, d=128, bs=16, nb=200, bst=8 * 2048, hst=2048,
          dtype=BF16, cdtype=BF16, ws=P, wsb=1 << 30, stream=None)


@pytest.mark.parametrize("over,code,needle", [
    (dict(dtype=FP8), UNS, "dtype"), (dict(cdtype=F32), UNS, "differs"), (dict(cdtype=FP8), INV, "k_scale"),
    (dict(d=80), UNS, "no kernel"), (dict(n=-1), INV, "num_seqs"), (dict(mq=-1), INV, "max_query_len"),
    (dict(rows=-1), INV, "total_query_rows"), (dict(h=12), INV, "multiple of"),
    (dict(n=70000), UNS, "65535"), (dict(mc=1 << 29, bts=1 << 26), UNS, "exceeds"),
    (dict(mq=1 << 30), UNS, "too many"), (dict(sc=None), INV, "non-null"), (dict(q=None), INV, "non-null"),
    (dict(bt=None), INV, "non-null"), (dict(cl=None), INV, "non-null"), (dict(q=P + 2), INV, "misaligned"),
    (dict(sc=P + 2), INV, "misaligned"), (dict(bts=31), INV, "too small"), (dict(sh=499), INV, "overlap"),
    (dict(ss=8 * 512 - 1), INV, "overlap"), (dict(ws=None), WS, "bytes needed"),
    (dict(wsb=ws_bytes(9, 16, 500) - 1), WS, "bytes needed"), (dict(ws=P + 16), INV, "256-byte"),
])
def test_weights_rejects(over, code, needle):
    refused("vpa_paged_attention_weights", WT, over, code, needle)


@pytest.mark.parametrize("over", [dict(n=0), dict(mq=0), dict(mc=0), dict(rows=0)])
def test_weights_of_nothing(over):
    assert call("vpa_paged_attention_weights", WT, {**over, "sc": None, "ws": None})[0] == 0


def test_weights_workspace_covers_rows_and_chunks():
    assert ws_bytes(0, 16, 5) == ws_bytes(4, 0, 5) == ws_bytes(4, 16, 0) == 0
    # every row's logits up to a whole chunk, and a pair per chunk
    assert ws_bytes(4, 16, 257) >= 4 * 16 * (512 * 4 + 2 * 8)
    assert ws_bytes(1 << 20, 64, 1 << 17) > 1 << 40  # in 64 bits


EV = dict(kc=P, vc=P, sc=P, ss=8 * 512, sh=512, bt=P, bts=32, cl=P, new=2 * P, kept=P, n=4, mc=500,
          budget=64, first=4, last=8, kvh=8, d=128, bs=16, nb=200, bst=8 * 2048, hst=2048, cdtype=BF16,
          ws=P, wsb=1 << 20, stream=None)


def ews_bytes(n, kvh, ctx, bs):
    return _lib.load().vpa_evict_kv_cache_workspace_size(n, kvh, ctx, bs)


@pytest.mark.parametrize("over,code,needle", [
    (dict(ws=None), WS, "bytes needed"), (dict(wsb=ews_bytes(4, 8, 500, 16) - 1), WS, "bytes needed"),
    (dict(ws=P + 64), INV, "256-byte"),
    (dict(cdtype=7), UNS, "dtype"), (dict(d=80), UNS, "no kernel"), (dict(n=-1), INV, "num_seqs"),
    (dict(budget=0), INV, "budget"), (dict(budget=-3), INV, "budget"), (dict(first=-1), INV, "budget"),
    (dict(last=-1), INV, "budget"), (dict(first=60, last=5), INV, "budget"),
    (dict(first=2 ** 31 - 1, last=2 ** 31 - 1), INV, "budget"), (dict(sc=None), INV, "non-null"),
    (dict(kept=None), INV, "non-null"), (dict(new=None), INV, "non-null"), (dict(new=P, cl=P), INV, "must not"),
    (dict(bts=31), INV, "too small"), (dict(sh=499), INV, "overlap"), (dict(ss=100), INV, "overlap"),
    (dict(n=1 << 20), UNS, "2^18"), (dict(vc=None), INV, "non-null"), (dict(kc=P + 4), INV, "aligned"),
])
def test_evict_rejects(over, code, needle):
    refused("vpa_evict_kv_cache", EV, over, code, needle)


def vws(b, k, v):
    return _lib.load().vpa_verify_draft_tokens_workspace_size(b, k, v)


VE = dict(ids=P, cnt=P, t=P, ts=5 * 1000, tr=1000, d=P, ds=4000, dr=1000, di=P, nd=None, temp=None, au=P,
          su=P, b=3, k=4, v=1000, dtype=BF16, ws=P, wsb=1 << 30, stream=None)


@pytest.mark.parametrize("over,code,needle", [
    (dict(dtype=FP8), UNS, "dtype"), (dict(b=-1), INV, "num_seqs"), (dict(k=-1), INV, "max_drafts"),
    (dict(v=-1), INV, "vocab"), (dict(v=0), INV, "empty rows"), (dict(k=65), UNS, "exceeds 64"),
    (dict(b=65536), UNS, "65535"), (dict(b=65535, k=64, v=1 << 24), UNS, "too many logits"),
    (dict(ids=None), INV, "non-null"), (dict(cnt=None), INV, "non-null"), (dict(t=None), INV, "non-null"),
    (dict(di=None), INV, "non-null"), (dict(au=None), INV, "non-null"), (dict(su=None), INV, "non-null"),
    (dict(ts=-1), INV, "negative"), (dict(t=P + 1), INV, "misaligned"), (dict(d=P + 1), INV, "misaligned"),
    (dict(ws=None), WS, "bytes needed"), (dict(wsb=vws(3, 4, 1000) - 1), WS, "bytes needed"),
    (dict(ws=P + 128), INV, "256-byte"),
])
def test_verify_rejects(over, code, needle):
    refused("vpa_verify_draft_tokens", VE, over, code, needle)


def test_verify_of_no_sequences():
    assert call("vpa_verify_draft_tokens", VE, dict(b=0, ids=None, ws=None))[0] == 0
    assert vws(0, 4, 10) == vws(4, -1, 10) == vws(4, 4, 0) == 0


def test_sizes_hold_their_arguments():
    """The ctypes signatures carry 64-bit strides and counts."""
    sig = _lib.SIGNATURES
    assert sig["vpa_paged_attention_weights"][1].count(ctypes.c_int64) == 6
    assert sig["vpa_verify_draft_tokens"][1].count(ctypes.c_int64) == 4


def test_frequencies():
    f, a = vpa.rotary_frequencies(8, 10000.0, "cpu")
    assert f.dtype == torch.float64 and f.tolist() == [1.0, 10000.0 ** -0.25, 10000.0 ** -0.5,
                                                       10000.0 ** -0.75]
    assert a.tolist() == [0, 0, 0, 0]
    _, a = vpa.rotary_frequencies(20, 1e4, "cpu", sections=(5, 3, 2))
    assert a.tolist() == [0] * 5 + [1] * 3 + [2] * 2
    _, a = vpa.rotary_frequencies(20, 1e4, "cpu", sections=(5, 3, 2), interleaved=True)
    assert a.tolist() == [0, 1, 2, 0, 1, 2, 0, 1, 0, 0]
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, sections=(2, 1)),
                dict(rotary_dim=8, sections=(5, -1))):
        with pytest.raises(vpa.VpaError):
            vpa.rotary_frequencies(theta=1e4, device="cpu", **bad)


def test_wrappers_refuse_host_tensors():
    z = torch.zeros(2, 2, 64)
    f, a = vpa.rotary_frequencies(64, 1e4, "cpu")
    pos = torch.zeros(1, 2, dtype=torch.int64)
    with pytest.raises(vpa.VpaError, match="GPU only"):
        vpa.rotary_qk(z, z, pos, f, a)
    kc, vc = torch.zeros(2, 2, 16, 16, 4), torch.zeros(2, 2, 64, 16)
    u = torch.zeros(2, 1, dtype=torch.uint32)
    with pytest.raises(vpa.VpaError, match="GPU only"):
        vpa.evict_kv_cache(kc, vc, z, u, u[:, 0], 4)
    with pytest.raises(vpa.VpaError, match="GPU only"):
        vpa.paged_attention_weights(z, kc, None, u, u[:, 0], 1.0, z)
    with pytest.raises(vpa.VpaError, match="GPU only"):
        vpa.verify_draft_tokens(z, u, u, u)
