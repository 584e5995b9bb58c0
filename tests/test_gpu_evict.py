"""GPU tests of evict_kv_cache: kept tokens, moved caches and scores, all exact
(nothing is computed but comparisons)."""

import numpy as np
import pytest
import torch

import vpa
from tests import _loop_oracle as ref
from tests._util import block_tables_for, u32

pytestmark = pytest.mark.gpu

WORD = {1: torch.uint8, 2: torch.int16, 4: torch.int32}


def problem(device, elem, kvh, d, bs, lens, seed=0, scores=None, pad_cols=1, extra=3):
    """Caches of random bytes (as the words of an element type)."""
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens)
    nb = int((-(-lens // bs)).sum()) + 5
    tables = block_tables_for(rng, list(lens), nb, bs, pad_cols=pad_cols)
    x = 16 // elem
    kind = {1: np.uint8, 2: np.int16, 4: np.int32}[elem]
    info = np.iinfo(kind)
    kc = rng.integers(info.min, info.max, (nb, kvh, d // x, bs, x), dtype=kind, endpoint=True)
    vc = rng.integers(info.min, info.max, (nb, kvh, d, bs), dtype=kind, endpoint=True)
    width = tables.shape[1] * bs + extra
    if scores is None:
        scores = np.exp(1.5 * rng.standard_normal((len(lens), kvh, width))).astype(np.float32)
    return dict(kc=kc, vc=vc, tables=tables, lens=lens, scores=scores, elem=elem)


def dev(a, device, elem):
    t = torch.from_numpy(a.copy()).to(device)
    return t if elem == 1 else t.view(torch.bfloat16 if elem == 2 else torch.float32)


def run(device, p, budget, first=0, last=0, **kw):
    kc, vc = dev(p["kc"], device, p["elem"]), dev(p["vc"], device, p["elem"])
    sc = torch.from_numpy(p["scores"].copy()).to(device)
    new, kept = vpa.evict_kv_cache(kc, vc, sc, u32(p["tables"], device), u32(p["lens"], device),
                                   budget, keep_first=first, keep_last=last, **kw)
    torch.cuda.synchronize()
    words = lambda t: t.cpu().view(WORD[p["elem"]]).numpy()  # noqa: E731
    return words(kc), words(vc), sc.cpu().numpy(), new.cpu().numpy(), kept.cpu().numpy()


def check(p, got, budget, first=0, last=0, lens=None):
    kc, vc, sc, new, kept = got
    lens = p["lens"] if lens is None else lens
    want_new, want = ref.evict(p["scores"], lens, budget, first, last)
    assert np.array_equal(new, want_new)
    for s in range(len(lens)):
        for j in range(kept.shape[1]):
            n = len(want[s][j])
            assert np.array_equal(kept[s, j, :n], want[s][j]), (s, j)
            assert np.all(kept[s, j, n:] == 0xFFFFFFFF)
            exp = p["scores"][s, j].copy()
            if lens[s] > budget:
                exp[:lens[s]] = 0
                exp[:n] = p["scores"][s, j][want[s][j]]
            assert np.array_equal(sc[s, j].view(np.int32), exp.view(np.int32))
    assert np.array_equal(kc, ref.moved(p["kc"], p["tables"], want, True))
    assert np.array_equal(vc, ref.moved(p["vc"], p["tables"], want, False))


@pytest.mark.parametrize("elem", [1, 2, 4])
@pytest.mark.parametrize("bs", [8, 16, 32])
@pytest.mark.parametrize("d", [64, 96, 128, 192, 256])
def test_types_and_shapes(device, elem, bs, d):
    p = problem(device, elem, 3, d, bs, [300, 97, 700, 64, 65, 1, 0], seed=bs + d)
    check(p, run(device, p, 64, 4, 16), 64, 4, 16)


@pytest.mark.parametrize("budget,first,last", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (7, 3, 4), (50, 0, 0),
                                               (50, 50, 0), (50, 0, 50), (255, 4, 32), (256, 4, 32),
                                               (257, 0, 1), (999, 0, 0), (1000, 8, 8), (5000, 1, 1)])
def test_budgets(device, budget, first, last):
    p = problem(device, 2, 2, 64, 16, [1000, 1001, 50, 51, 2, 1, 0, 300], seed=budget)
    check(p, run(device, p, budget, first, last), budget, first, last)


def test_ties_nan_infinities_zeros(device):
    rng = np.random.default_rng(1)
    lens = [900, 900, 900, 900, 900, 900]
    p = problem(device, 2, 2, 64, 16, lens, seed=2)
    sc = p["scores"]
    sc[0] = 1.0                                                  # all equal: the first ones
    sc[1] = rng.integers(0, 3, sc[1].shape)                      # many ties at the border
    sc[2] = rng.choice(np.array([0.0, -0.0], np.float32), sc[2].shape)  # equal zeros
    sc[3] = np.where(rng.random(sc[3].shape) < 0.4, np.nan, sc[3])
    sc[4] = rng.choice(np.array([np.inf, -np.inf, np.nan, 0, -1, 1e-45, -1e-45, 3e38],
                                np.float32), sc[4].shape)
    sc[5] = np.nan
    for budget in (100, 500, 890):
        check(p, run(device, p, budget, 4, 9), budget, 4, 9)


def test_negative_and_close_scores(device):
    """Neighbouring floats and both signs."""
    rng = np.random.default_rng(3)
    p = problem(device, 2, 4, 64, 16, [2000], seed=3)
    base = rng.integers(0, 40, p["scores"].shape).astype(np.uint32) + np.uint32(0x3F800000)
    sign = rng.integers(0, 2, p["scores"].shape).astype(np.uint32) << np.uint32(31)
    p["scores"] = (base | sign).view(np.float32)
    check(p, run(device, p, 777, 0, 0), 777)


def test_long_sequence(device):
    """More tokens than a pass of the workgroup, a sparse choice and a dense one."""
    p = problem(device, 1, 2, 64, 32, [20000, 5], seed=4)
    check(p, run(device, p, 300, 4, 64), 300, 4, 64)
    check(p, run(device, p, 19000, 4, 64), 19000, 4, 64)


@pytest.mark.parametrize("elem,bs,d", [(1, 8, 64), (2, 16, 128), (2, 8, 96), (4, 32, 64)])
@pytest.mark.parametrize("budget,first,last", [(5, 0, 0), (40, 1, 3), (300, 260, 20)])
def test_most_columns_empty(device, elem, bs, d, budget, first, last):
    """Few tokens stay of contexts of several table windows and of one: whole stretches
    of columns, and whole windows, keep nothing."""
    lens = [600 * bs + 5, 1100 * bs + 1, 511 * bs + 3, 512 * bs, 40 * bs]
    p = problem(device, elem, 2, d, bs, lens, seed=budget + d)
    p["scores"][1, 0, 20 * bs:] = 0.0    # nothing behind but the last
    p["scores"][0, 1, :560 * bs] = -1.0  # nothing before
    check(p, run(device, p, budget, first, last), budget, first, last)
    got = run(device, p, budget, first, last, max_context_len=512 * bs)
    check(p, got, budget, first, last, lens=np.minimum(lens, 512 * bs))


def test_already_sorted_prefix_stays(device):
    """The highest scores in front: nothing moves; in the back: everything does."""
    p = problem(device, 2, 2, 128, 16, [1500, 1500], seed=5)
    w = p["scores"].shape[2]
    p["scores"][0] = np.arange(w, 0, -1)
    p["scores"][1] = np.arange(w)
    got = run(device, p, 600)
    check(p, got, 600)


def test_max_context_len_clamps(device):
    p = problem(device, 2, 2, 64, 16, [500, 90], seed=6)
    got = run(device, p, 80, 2, 3, max_context_len=200)
    check(p, got, 80, 2, 3, lens=np.minimum(p["lens"], 200))


def test_absent_blocks_are_left_alone(device):
    """Table entries past the pool: their tokens are neither read nor written, the
    others move as ever."""
    p = problem(device, 2, 2, 64, 16, [200, 120], seed=7)
    nb = p["kc"].shape[0]
    p["tables"][0, 2] = nb + 3
    p["tables"][0, 7] = 0xFFFFFFFF
    kc, vc, sc, new, kept = run(device, p, 96, 4, 8)
    want_new, want = ref.evict(p["scores"], p["lens"], 96, 4, 8)
    assert np.array_equal(new, want_new)
    ek, ev = p["kc"].copy(), p["vc"].copy()
    for s in range(2):
        for j in range(2):
            assert np.array_equal(kept[s, j], want[s][j])
            for to, at in enumerate(want[s][j]):
                sb, db = int(p["tables"][s, at // 16]), int(p["tables"][s, to // 16])
                if sb < nb and db < nb:
                    ek[db, j, :, to % 16] = p["kc"][sb, j, :, at % 16]
                    ev[db, j, :, to % 16] = p["vc"][sb, j, :, at % 16]
    assert np.array_equal(kc, ek) and np.array_equal(vc, ev)


def test_strided_caches_and_scores(device):
    p = problem(device, 2, 2, 64, 16, [333, 40], seed=8)
    nb = p["kc"].shape[0]
    pool_k = torch.zeros((nb, 4, 8, 16, 8), dtype=torch.bfloat16, device=device)
    pool_v = torch.zeros((nb, 4, 64, 16), dtype=torch.bfloat16, device=device)
    pool_k[:, 1:3] = dev(p["kc"], device, 2)
    pool_v[:, 1:3] = dev(p["vc"], device, 2)
    wide = torch.full((2, 4, p["scores"].shape[2] + 9), 7.0, device=device)
    sc = wide[:, 1:3, 4:-5]
    sc.copy_(torch.from_numpy(p["scores"]))
    new, kept = vpa.evict_kv_cache(pool_k[:, 1:3], pool_v[:, 1:3], sc, u32(p["tables"], device),
                                   u32(p["lens"], device), 100, keep_first=1, keep_last=2)
    got = (pool_k[:, 1:3].contiguous().cpu().view(torch.int16).numpy(),
           pool_v[:, 1:3].contiguous().cpu().view(torch.int16).numpy(), sc.contiguous().cpu().numpy(),
           new.cpu().numpy(), kept.cpu().numpy())
    check(p, got, 100, 1, 2)
    assert not pool_k[:, ::3].any() and not pool_v[:, ::3].any()
    assert (wide[:, 0] == 7).all() and (wide[:, 3] == 7).all() and (wide[..., :4] == 7).all()


def test_no_sequences(device):
    p = problem(device, 2, 2, 64, 16, [40], seed=9)
    kc, vc = dev(p["kc"], device, 2), dev(p["vc"], device, 2)
    new, kept = vpa.evict_kv_cache(kc, vc, torch.zeros((0, 2, 64), device=device),
                                   u32(p["tables"][:0], device), u32(p["lens"][:0], device), 8)
    assert new.shape == (0,) and kept.shape == (0, 2, 8)


def test_graph_replays(device):
    p = problem(device, 2, 2, 64, 16, [600, 300, 90], seed=10)
    bt, cl = u32(p["tables"], device), u32(p["lens"], device)
    kc, vc = dev(p["kc"], device, 2), dev(p["vc"], device, 2)
    sc = torch.from_numpy(p["scores"].copy()).to(device)
    new = torch.empty(3, dtype=torch.uint32, device=device)
    kept = torch.empty((3, 2, 128), dtype=torch.uint32, device=device)

    def step(kc, vc, sc, new, kept):
        vpa.evict_kv_cache(kc, vc, sc, bt, cl, 128, keep_first=4, keep_last=16, max_context_len=600,
                           new_context_lens=new, kept=kept)

    step(kc.clone(), vc.clone(), sc.clone(), new, kept)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(kc, vc, sc, new, kept)
    for i in range(3):
        cl.copy_(u32([600 - i, 300 + i, 90 + 30 * i], device))
        sc.uniform_()
        mine = [kc.clone(), vc.clone(), sc.clone(), torch.empty_like(new), torch.empty_like(kept)]
        step(*mine)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(mine, (kc, vc, sc, new, kept)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
