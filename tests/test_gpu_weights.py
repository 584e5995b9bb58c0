"""GPU tests of paged_attention_weights against the 64-bit restatement.

A weight p = exp(l - m) / S of a row. The logit l (natural units) is a sum of D products in
f32: off by at most (D + 3) u sum|q k| scale, u = 2^-24 (16-bit products are exact
in f32; the matrix cores add in f32), which the tests bound through the
largest |q|.|k| of the problem; p is then off by twice that relatively (its own
exponential and the sum's), plus the exponentials' 4 u each, the product with log2 e (|l| u)
and the chunks' merging (below 16 u). Weights of a score add up, in f32: (rows * G + 1) u
of the score."""

import itertools

import numpy as np
import pytest
import torch

import vpa
from tests import _loop_oracle as ref
from tests._util import block_tables_for, u32

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
KS = 0.013


def np64(t):
    return t.detach().double().cpu().numpy()


def problem(device, dtype, fp8, d, bs, h, kvh, lens, rows=None, seed=0, extra=5, scale_q=1.0):
    rng = np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    lens = np.asarray(lens)
    nb = int((-(-lens // bs)).sum()) + 7
    tables = block_tables_for(rng, list(lens), nb, bs, pad_cols=1)
    if fp8:
        kc = (torch.randn((nb, kvh, d // 16, bs, 16), generator=gen) / KS).clamp(-448, 448).to(
            torch.float8_e4m3fn)
        keys = kc.float().double().numpy() * np.float64(np.float32(KS))
        kc = kc.view(torch.uint8)
    else:
        x = 128 // torch.finfo(dtype).bits
        kc = torch.randn((nb, kvh, d // x, bs, x), generator=gen).to(dtype)
        keys = np64(kc)
    n = np.ones(len(lens), int) if rows is None else np.asarray(rows)
    q = (scale_q * torch.randn((int(n.sum()), h, d), generator=gen)).to(dtype)
    width = tables.shape[1] * bs + extra
    scores = torch.rand((len(lens), kvh, width), generator=gen)
    cu = None if rows is None else np.concatenate([[0], np.cumsum(n)]).astype(np.uint32)
    return dict(q=q.to(device), kc=kc.to(device), keys=keys, tables=tables, lens=lens, cu=cu,
                scores=scores.to(device), ks=torch.tensor([KS], device=device) if fp8 else None,
                h=h, kvh=kvh, d=d)


def run(device, p, causal=True, scale=None, **kw):
    scale = p["d"] ** -0.5 if scale is None else scale
    got = p["scores"].clone()
    vpa.paged_attention_weights(p["q"], p["kc"], p["ks"], u32(p["tables"], device),
                                u32(p["lens"], device), scale, got,
                                cu_seqlens_q=None if p["cu"] is None else u32(p["cu"], device),
                                causal=causal, **kw)
    return got


def check(p, got, causal=True, scale=None, lens=None):
    scale = p["d"] ** -0.5 if scale is None else scale
    lens = p["lens"] if lens is None else lens
    want = ref.attention_weights(np64(p["q"]), p["keys"], p["tables"], lens, scale,
                                 np64(p["scores"]), p["cu"], causal)
    size = scale * np.nanmax(np.abs(np64(p["q"])).sum(-1)) * np.nanmax(np.abs(p["keys"]))
    rows = 1 if p["cu"] is None else int(np.diff(p["cu"].astype(int)).max())
    rel = 2 * (p["d"] + 3) * U * size + (24 + 2 * size) * U
    tol = (want - np64(p["scores"])) * rel + want * (rows * p["h"] // p["kvh"] + 2) * U
    err = np.abs(np64(got) - want)
    assert np.all(err <= tol), (err / np.maximum(tol, 1e-300)).max()
    for s, n in enumerate(lens):  # behind the context nothing changes
        assert torch.equal(got[s, :, int(n):], p["scores"][s, :, int(n):])


COMBOS = [(torch.bfloat16, False), (torch.float16, False), (torch.float32, False),
          (torch.bfloat16, True), (torch.float16, True), (torch.float32, True)]


@pytest.mark.parametrize("dtype,fp8", COMBOS)
@pytest.mark.parametrize("d,bs", list(itertools.product([64, 96, 128, 192, 256], [8, 16, 32])))
def test_decode_rows(device, dtype, fp8, d, bs):
    p = problem(device, dtype, fp8, d, bs, 6, 3, [1, 17, 255, 256, 257, 700], seed=d + bs)
    check(p, run(device, p))


@pytest.mark.parametrize("dtype,fp8", COMBOS)
@pytest.mark.parametrize("d,bs", [(64, 8), (96, 32), (128, 16), (192, 8), (256, 32)])
def test_longer_contexts(device, dtype, fp8, d, bs):
    """Contexts that are split over workgroups, in two launches."""
    p = problem(device, dtype, fp8, d, bs, 6, 3, [1, 769, 0, 1500], seed=d + bs + 1)
    check(p, run(device, p))


@pytest.mark.parametrize("dtype,fp8,d", [(torch.bfloat16, False, 128), (torch.float32, False, 64),
                                         (torch.float16, True, 96), (torch.float32, True, 192)])
def test_thousands_of_pairs(device, dtype, fp8, d):
    """2048 (sequence, kv head) pairs and more, more sequences than are ordered."""
    rng = np.random.default_rng(d)
    lens = rng.integers(0, 70, size=515)
    lens[300] = 333
    p = problem(device, dtype, fp8, d, 16, 8, 4, lens, seed=24)
    check(p, run(device, p))
    short = np.minimum(lens, 500)[:512]
    p = problem(device, dtype, fp8, d, 16, 4, 4, short, seed=25)
    check(p, run(device, p))


@pytest.mark.parametrize("h,kvh", [(16, 8), (8, 8), (14, 2), (32, 1), (40, 2), (3, 1)])
@pytest.mark.parametrize("dtype,fp8", COMBOS[:4])
def test_groups(device, dtype, fp8, h, kvh):
    p = problem(device, dtype, fp8, 128, 16, h, kvh, [33, 1030], seed=h)
    check(p, run(device, p))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,fp8", COMBOS)
def test_several_rows(device, dtype, fp8, causal):
    """Ragged rows: none, one, several, more than a row tile of 16 and of 64; a
    sequence that has fewer tokens than rows (its first rows see nothing)."""
    p = problem(device, dtype, fp8, 64, 16, 4, 2, [40, 300, 600, 17, 5, 64], rows=[0, 1, 40, 17, 9, 8],
                seed=11)
    check(p, run(device, p, causal), causal)


@pytest.mark.parametrize("dtype,fp8,d,bs", [(torch.bfloat16, False, 128, 16),
                                            (torch.float32, False, 64, 8),
                                            (torch.float16, True, 96, 32),
                                            (torch.float32, True, 256, 16)])
@pytest.mark.parametrize("causal", [True, False])
def test_many_sequences(device, dtype, fp8, d, bs, causal):
    """512 and more (sequence, kv head) pairs: contexts in one launch, the longest first;
    ragged rows and lengths, some of them none."""
    rng = np.random.default_rng(d)
    lens = rng.integers(0, 150, size=131)
    lens[[3, 77]] = [700, 1]
    rows = np.minimum(rng.integers(0, 4, size=131), np.maximum(lens, 1))
    p = problem(device, dtype, fp8, d, bs, 8, 4, lens, rows=rows, seed=21)
    check(p, run(device, p, causal), causal)


def test_more_sequences_than_are_ordered(device):
    rng = np.random.default_rng(5)
    p = problem(device, torch.bfloat16, False, 64, 16, 1, 1, rng.integers(0, 90, size=601), seed=22)
    check(p, run(device, p))


@pytest.mark.parametrize("dtype,fp8,d", [(torch.bfloat16, False, 64), (torch.float32, False, 64),
                                         (torch.bfloat16, True, 192)])
def test_many_rows_of_many_sequences(device, dtype, fp8, d):
    """Chunks of several pieces, blocks of rows that are not full."""
    rng = np.random.default_rng(6)
    lens = rng.integers(1, 1100, size=48)
    lens[0] = 2100
    rows = np.minimum(rng.integers(0, 12, size=48), lens)
    p = problem(device, dtype, fp8, d, 16, 18, 6, lens, rows=rows, seed=23)
    check(p, run(device, p))


def test_sum_of_weights(device):
    """Every row's weights sum to 1: 40 additions of 600 values, f32."""
    p = problem(device, torch.bfloat16, False, 128, 16, 16, 8, [600, 1, 4096], seed=1)
    p["scores"].zero_()
    got = run(device, p).sum(-1)
    assert torch.allclose(got, torch.full_like(got, 2.0), rtol=0, atol=2 * 4200 * U)


def test_empty_sequences_and_clamps(device):
    p = problem(device, torch.bfloat16, False, 128, 16, 8, 4, [0, 5, 0, 300], seed=2)
    check(p, run(device, p))
    # max_context_len clamps the lengths
    got = run(device, p, max_context_len=100)
    check(p, got, lens=np.minimum(p["lens"], 100))
    # no sequence at all
    e = torch.zeros((0, 4, 8), device=device)
    vpa.paged_attention_weights(p["q"][:0], p["kc"], None, u32(p["tables"][:0], device),
                                u32(p["lens"][:0], device), 1.0, e)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_stale_tokens_and_absent_blocks(device, dtype):
    """NaN and infinities behind the context in its last block, and in blocks the
    tables do not name, leave no trace; a table entry past the pool has no tokens."""
    p = problem(device, dtype, False, 128, 16, 8, 4, [20, 100, 37], seed=3)
    clean = run(device, p)
    nb = p["kc"].shape[0]
    bad = torch.ones(nb, 16, dtype=torch.bool)
    for s, n in enumerate(p["lens"]):
        for t in range(int(n)):
            bad[int(p["tables"][s, t // 16]), t % 16] = False
    kc = p["kc"].permute(0, 3, 1, 2, 4)
    kc[bad.to(device)] = float("nan")
    p["kc"].permute(0, 3, 1, 2, 4)[0] = float("inf")
    assert torch.equal(run(device, p), clean)
    p["tables"][1, 2] = nb + 5
    p["tables"][2, :] = 0xFFFFFFFF
    p["keys"] = np.nan_to_num(p["keys"])
    check(p, run(device, p))


def test_nan_query_marks_its_own_scores_only(device):
    p = problem(device, torch.bfloat16, False, 128, 16, 8, 4, [50, 70], seed=4)
    clean = run(device, p)
    p["q"][1, 3, 5] = float("nan")
    got = run(device, p)
    assert torch.isnan(got[1, 1, :70]).all()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[1, 1, :70] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 9, 33])
def test_infinite_keys(device, dtype, rows):
    """A key of -inf against positive queries has weight 0, whatever rows share its tile."""
    p = problem(device, dtype, False, 64, 16, 4, 2, [300, 40], rows=[rows, rows], seed=9)
    p["q"][..., 3] = p["q"][..., 3].abs() + 1
    blk = int(p["tables"][0, 2])
    x = p["kc"].shape[-1]
    p["kc"][blk, :, 3 // x, 7, 3 % x] = float("-inf")
    p["keys"][blk, :, 3 // x, 7, 3 % x] = -np.inf
    got = run(device, p)
    assert torch.equal(got[0, :, 39], p["scores"][0, :, 39])
    p["keys"][blk, :, 3 // x, 7, 3 % x] = -1e6  # (as far as exp is concerned)
    size = np64(p["q"])
    want = ref.attention_weights(size, p["keys"], p["tables"], p["lens"], 0.125, np64(p["scores"]),
                                 p["cu"], True)
    p["keys"][blk, :, 3 // x, 7, 3 % x] = 0  # the bound is that of the finite keys
    rel = 2 * 67 * U * 0.125 * np.abs(size).sum(-1).max() * np.abs(p["keys"]).max()
    rel += (24 + 2 * 0.125 * np.abs(size).sum(-1).max() * np.abs(p["keys"]).max()) * U
    tol = (want - np64(p["scores"])) * rel + want * (rows * 2 + 2) * U
    assert np.all(np.abs(np64(got) - want) <= tol)


def test_longest_context_held_in_one_workgroup(device):
    """512 pairs of one row each, the logits of 16384 tokens in LDS; one token more takes
    two launches."""
    lens = np.full(64, 5)
    lens[40] = 16384
    p = problem(device, torch.bfloat16, False, 64, 32, 8, 8, lens, seed=10)
    check(p, run(device, p))
    wide = np.concatenate([p["tables"], np.zeros((64, 1), np.uint32)], 1)
    a = dict(p, tables=wide, scores=torch.nn.functional.pad(p["scores"], (0, 32)))
    got = run(device, a, max_context_len=16385)
    check(a, got)


def test_large_logits(device):
    """Logits of several hundred: one weight takes it all."""
    p = problem(device, torch.float32, False, 64, 16, 4, 2, [500, 3], seed=5, scale_q=40.0)
    check(p, run(device, p, scale=0.5), scale=0.5)


def test_strided_scores_and_repeatability(device):
    p = problem(device, torch.float16, False, 128, 32, 16, 4, [1000, 64, 333], seed=6)
    a = run(device, p)
    assert torch.equal(a, run(device, p))
    wide = torch.zeros((3, 6, p["scores"].shape[2] + 11), device=device)
    view = wide[:, 1:5, 3:-8]
    view.copy_(p["scores"])
    vpa.paged_attention_weights(p["q"], p["kc"], None, u32(p["tables"], device),
                                u32(p["lens"], device), 128 ** -0.5, view)
    assert torch.equal(view, a)
    assert not wide[:, 0].any() and not wide[:, 5].any() and not wide[:, :, :3].any()


def test_graph_and_stream(device):
    p = problem(device, torch.bfloat16, False, 128, 16, 16, 8, [400, 90, 1], seed=7)
    bt, cl = u32(p["tables"], device), u32(p["lens"], device)
    sc = p["scores"].clone()
    ws = vpa.paged_attention_weights_workspace(3, 16, 512, device)

    def step(scores):
        vpa.paged_attention_weights(p["q"], p["kc"], None, bt, cl, 128 ** -0.5, scores,
                                    max_context_len=400, workspace=ws)

    step(sc.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(sc)
    want = sc.clone()
    for i in range(3):
        p["q"].normal_()
        cl.copy_(u32([400 - i, 90 - 7 * i, i], device))
        step(want)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(sc, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        vpa.paged_attention_weights(p["q"], p["kc"], None, bt, cl, 128 ** -0.5, sc,
                                    max_context_len=400)
    step(want)
    torch.cuda.synchronize()
    assert torch.equal(sc, want)
