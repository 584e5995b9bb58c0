"""Refusals of the block-scaled cache's, the shared blocks' and the logits' entry points, on
the host before any launch (no GPU here), and their Python wrappers' checks."""

import ctypes

import pytest
import torch

import vpa
from tests.test_loop_abi import call, refused
from vpa import _lib

INV, UNS, WS = (_lib.VPA_ERR_INVALID_ARGUMENT, _lib.VPA_ERR_UNSUPPORTED, _lib.VPA_ERR_WORKSPACE)
P = 1 << 20  # 256-byte aligned non-null host value standing in for a device pointer
BF16, F32, FP8 = _lib.DTYPE_BF16, _lib.DTYPE_F32, _lib.DTYPE_FP8_E4M3

AP = dict(k=P, v=P, kst=1024, vst=1024, ks=P, vs=P, sst=8, kc=P, vc=P, slots=P, t=4, kvh=8, d=128,
          bs=16, nb=10, bst=8 * 2048, hst=2048, dtype=BF16, stream=None)


@pytest.mark.parametrize("over,code,needle", [
    (dict(dtype=FP8), UNS, "dtype"), (dict(dtype=9), UNS, "dtype"), (dict(t=-1), INV, "num_tokens"),
    (dict(d=80), UNS, "no kernel"), (dict(bs=24), UNS, "no kernel"), (dict(nb=0), INV, "positive"),
    (dict(hst=100), INV, "strides"), (dict(kc=None), INV, "non-null"), (dict(vc=P + 8), INV, "aligned"),
    (dict(ks=None), INV, "key_scales"), (dict(vs=None), INV, "value_scales"),
    (dict(ks=P + 2), INV, "aligned"), (dict(sst=7), INV, "scale_block_stride"),
    (dict(k=None), INV, "non-null"), (dict(v=None), INV, "non-null"), (dict(slots=None), INV, "non-null"),
    (dict(kst=1000), INV, "token stride"), (dict(vst=1000), INV, "token stride"),
    (dict(k=P + 8), INV, "16-byte"), (dict(kst=1028), INV, "16-byte"),
    (dict(t=1 << 26), INV, "too many"), (dict(t=1 << 62), INV, "too many"),
])
def test_append_rejects(over, code, needle):
    refused("vpa_reshape_and_cache_block_scaled", AP, over, code, needle)


def aws(n=4, mq=3, mc=20000, rows=9, h=16, kvh=8, d=128, dtype=BF16):
    return _lib.load().vpa_paged_attention_block_scaled_workspace_size(n, mq, mc, rows, h, kvh, d, dtype)


AT = dict(out=P, q=P, ks=P, vs=P, sst=8, kc=P, vc=P, bt=P, bts=1250, cu=P, cl=P, n=4, mq=3, mc=20000,
          rows=9, scale=0.1, eps=0.0, causal=1, h=16, kvh=8, d=128, bs=16, nb=200, bst=8 * 2048, hst=2048,
          dtype=BF16, ws=P, wsb=1 << 30, stream=None)


@pytest.mark.parametrize("over,code,needle", [
    (dict(dtype=FP8), UNS, "dtype"), (dict(d=80), UNS, "no kernel"), (dict(kc=None), INV, "non-null"),
    (dict(ks=None), INV, "key_scales"), (dict(sst=4), INV, "scale_block_stride"),
    (dict(n=-1), INV, "num_seqs"), (dict(mq=-1), INV, "max_query_len"), (dict(rows=-1), INV, "total"),
    (dict(mc=-1), INV, "max_context_len"), (dict(h=0), INV, "num_heads"), (dict(h=12), INV, "multiple of"),
    (dict(eps=-1.0), INV, "denom_eps"), (dict(eps=float("nan")), INV, "denom_eps"),
    (dict(eps=float("inf")), INV, "denom_eps"), (dict(mc=1 << 29, bts=1 << 26), UNS, "exceeds"),
    (dict(mq=1 << 30), UNS, "too many"), (dict(n=1 << 22, mc=1 << 16, bts=1 << 12), UNS, "too many"),
    (dict(out=None), INV, "non-null"), (dict(q=None), INV, "non-null"), (dict(bt=None), INV, "non-null"),
    (dict(cl=None), INV, "non-null"), (dict(q=P + 2), INV, "16-byte"), (dict(out=P + 8), INV, "16-byte"),
    (dict(bts=1249), INV, "too small"), (dict(ws=None), WS, "bytes needed"),
    (dict(wsb=aws() - 1), WS, "bytes needed"), (dict(ws=P + 16), INV, "256-byte"),
])
def test_attention_rejects(over, code, needle):
    refused("vpa_paged_attention_block_scaled", AT, over, code, needle)


def test_attention_of_nothing():
    for over in (dict(n=0), dict(mq=0), dict(rows=0)):
        assert call("vpa_paged_attention_block_scaled", AT, {**over, "out": None, "ws": None})[0] == 0


def test_attention_workspace():
    assert aws(n=0) == aws(mq=0) == aws(mc=0) == aws(rows=0) == aws(kvh=0) == 0
    assert aws(n=512, mc=4096, rows=512, mq=1) == aws(mc=512) == 0  # one chunk of keys: nothing to join
    # every row's parts: head_dim sums, a maximum and a sum
    assert aws() % (9 * 16 * 130 * 4) == 0 and aws() > 0
    assert aws(n=1, mq=1 << 20, mc=1 << 28, rows=1 << 20) >= 0  # in 64 bits


def buffers(n, base=P, stride=4096, size=4096):
    return ((ctypes.c_void_p * n)(*[base] * n), (ctypes.c_int64 * n)(*[stride] * n),
            (ctypes.c_int64 * n)(*[size] * n))


_b, _s, _z = buffers(3)
CP = dict(b=_b, s=_s, z=_z, n=3, src=P, dst=P, count=None, pairs=4, nb=10, stream=None)


@pytest.mark.parametrize("over,code,needle", [
    (dict(n=-1), INV, "num_buffers"), (dict(pairs=-1), INV, "max_pairs"), (dict(nb=-1), INV, "num_blocks"),
    (dict(b=None), INV, "non-null"), (dict(s=None), INV, "non-null"), (dict(z=None), INV, "non-null"),
    (dict(src=None), INV, "non-null"), (dict(dst=None), INV, "non-null"),
    (dict(b=buffers(3, base=0)[0]), INV, "buffer 0"), (dict(s=buffers(3, stride=4095)[1]), INV, "stride"),
    (dict(z=buffers(3, size=-1)[2]), INV, "stride"),
    (dict(s=buffers(3, stride=1 << 40)[1], z=buffers(3, size=1 << 31)[2]), INV, "2^31"),
])
def test_copy_rejects(over, code, needle):
    refused("vpa_copy_blocks", CP, over, code, needle)


def test_copy_of_nothing():
    assert call("vpa_copy_blocks", CP, dict(n=0, b=None))[0] == 0
    assert call("vpa_copy_blocks", CP, dict(pairs=0, src=None))[0] == 0


FK = dict(bt=P, bts=8, rb=P, pos=P, sh=P, nb=100, src=P, dst=P, n=4, ok=P, cs=P, cd=P, cc=P, ring=P,
          state=P, cap=100, bs=16, rows=6, stream=None)
STATE = [(dict(rows=-1), INV, "num_rows"), (dict(bts=-1), INV, "block_table_stride"),
         (dict(nb=0), INV, "num_blocks"), (dict(cap=0), INV, "free_ring_capacity"),
         (dict(bt=None), INV, "non-null"), (dict(rb=None), INV, "non-null"), (dict(ring=None), INV, "non-null"),
         (dict(state=None), INV, "non-null")]


@pytest.mark.parametrize("over,code,needle", STATE + [
    (dict(bs=0), INV, "block_size"), (dict(pos=None), INV, "positions"), (dict(sh=None), INV, "shared"),
    (dict(n=-1), INV, "num_forks"), (dict(n=1025), UNS, "1024"), (dict(src=None), INV, "src_rows"),
    (dict(dst=None), INV, "dst_rows"), (dict(ok=None), INV, "ok"), (dict(cs=None), INV, "copy_src"),
    (dict(cd=None), INV, "copy_dst"), (dict(cc=None), INV, "copy_count"),
])
def test_fork_rejects(over, code, needle):
    refused("vpa_fork_rows", FK, over, code, needle)


RL = dict(bt=P, bts=8, rb=P, sh=P, nb=100, keep=P, ring=P, state=P, cap=100, rows=6, stream=None)


@pytest.mark.parametrize("over,code,needle", STATE + [
    (dict(sh=None), INV, "shared"), (dict(keep=None), INV, "keep_blocks"),
    (dict(rows=1 << 16, bts=1 << 15), UNS, "2^31"),
])
def test_release_rejects(over, code, needle):
    refused("vpa_release_shared_blocks", RL, over, code, needle)


def test_release_of_no_rows():
    assert call("vpa_release_shared_blocks", RL, dict(rows=0, keep=None, bt=None, rb=None))[0] == 0


UN = dict(bt=P, bts=8, rb=P, pos=P, sh=P, nb=100, ok=P, cs=P, cd=P, cc=P, ring=P, state=P, cap=100, bs=16,
          rows=6, stream=None)


@pytest.mark.parametrize("over,code,needle", STATE + [
    (dict(bs=0), INV, "block_size"), (dict(pos=None), INV, "positions"), (dict(sh=None), INV, "shared"),
    (dict(ok=None), INV, "ok"), (dict(cs=None), INV, "copy_src"), (dict(cd=None), INV, "copy_dst"),
    (dict(cc=None), INV, "copy_count"),
])
def test_unshare_rejects(over, code, needle):
    refused("vpa_unshare_rows", UN, over, code, needle)


def cws(nb):
    return _lib.load().vpa_compact_blocks_workspace_size(nb)


CM = dict(bt=P, bts=8, rb=P, sh=None, nb=100, cs=P, cd=P, cc=P, ring=P, state=P, cap=100, rows=6, ws=P,
          wsb=1 << 20, stream=None)


@pytest.mark.parametrize("over,code,needle", STATE + [
    (dict(nb=1 << 31), UNS, "2^31"), (dict(cs=None), INV, "copy_src"), (dict(cd=None), INV, "copy_dst"),
    (dict(cc=None), INV, "copy_count"), (dict(ws=None), WS, "bytes needed"),
    (dict(wsb=cws(100) - 1), WS, "bytes needed"), (dict(ws=P + 64), INV, "256-byte"),
])
def test_compact_rejects(over, code, needle):
    refused("vpa_compact_blocks", CM, over, code, needle)


def test_compact_workspace():
    assert cws(0) == cws(-1) == 0 and cws(1) > 0
    # a bit per block and a count per 32 of them
    assert cws((1 << 31) - 1) >= 2 * (1 << 28)


AJ = dict(x=P, ss=3000, rs=1000, b=3, k1=3, v=1000, dtype=BF16, gen=P, gs=10, gl=P, pro=P, ps=20, pl=P, dr=P,
          rep=P, pres=P, freq=P, bi=P, bv=P, bst=5, bl=P, al=P, nm=4, aw=32, ar=P, stream=None)


@pytest.mark.parametrize("over,code,needle", [
    (dict(dtype=FP8), UNS, "dtype"), (dict(b=-1), INV, "num_seqs"), (dict(k1=-1), INV, "rows_per_seq"),
    (dict(v=-1), INV, "vocab"), (dict(gs=-1), INV, "generated_stride"), (dict(ps=-1), INV, "prompt_stride"),
    (dict(bst=-1), INV, "bias_stride"), (dict(nm=-1), INV, "num_masks"), (dict(aw=-1), INV, "allowed_stride"),
    (dict(gs=1 << 20), UNS, "2^20"), (dict(bst=1025), UNS, "1024"), (dict(x=None), INV, "non-null"),
    (dict(x=P + 1), INV, "misaligned"), (dict(rs=999), INV, "overlap"), (dict(ss=2999), INV, "overlap"),
    (dict(bi=None), INV, "go together"), (dict(bv=None), INV, "go together"),
    (dict(aw=31), INV, "allowed_stride"), (dict(ar=None), INV, "num_masks"),
    (dict(b=1 << 22, ss=1 << 40, v=1 << 20, rs=1 << 20, aw=1 << 15), UNS, "too many"),
])
def test_adjust_rejects(over, code, needle):
    refused("vpa_adjust_logits", AJ, over, code, needle)


def test_adjust_of_nothing():
    for over in (dict(b=0), dict(k1=0), dict(v=0)):
        assert call("vpa_adjust_logits", AJ, {**over, "x": None})[0] == 0


def test_wrappers_refuse_what_they_can_see():
    kc, vc = torch.zeros((2, 2, 4, 16, 16), dtype=torch.uint8), torch.zeros((2, 2, 64, 16), dtype=torch.uint8)
    s = torch.zeros((2, 2))
    u = torch.zeros((2, 1), dtype=torch.uint32)
    with pytest.raises(vpa.VpaError, match="GPU only"):
        vpa.reshape_and_cache_block_scaled(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), s, s, kc, vc,
                                           torch.zeros(1, dtype=torch.int64))
    with pytest.raises(vpa.VpaError, match="GPU only"):
        vpa.paged_attention_block_scaled(torch.zeros(2, 2, 64), s, s, kc, vc, u, u[:, 0], 1.0)
    with pytest.raises(vpa.VpaError, match="GPU only"):
        vpa.adjust_logits(torch.zeros(2, 8))
    with pytest.raises(vpa.VpaError, match="GPU only"):
        vpa.copy_blocks([s], u[:, 0], u[:, 0])
    a = vpa.DeviceBlockAllocator(8, 16, 2, 3, "cpu")
    assert a.shared is None
    a.enable_sharing()
    assert a.shared.dtype == torch.uint32 and a.shared.shape == (8,)
    with pytest.raises(vpa.VpaError, match="GPU only"):
        a.fork(u[:, 0], u[:, 0], [])
    with pytest.raises(vpa.VpaError, match="GPU only"):
        a.compact([])
