"""GPU tests of rotary_qk and rotary_reshape_and_cache against the 64-bit
restatement.

A value y = n_p cos a -+ n_s sin a is rounded once to its type (half a step,
finfo.eps / 2 of |y|). Before that, in f32 (u = 2^-24): the norm's sum of
squares takes at most 2 * 8 additions in a lane and 5 across lanes, its root,
quotient and product 5 more roundings, so n is off by at most 21 u / 2 + 5 u < 16 u;
sine and cosine by 4 u (angle remainder below pi / 4 in f32, series of 5 terms,
absolute), products and sum 2 u. Together below 24 u (|n_p| + |n_s|)."""

import itertools

import numpy as np
import pytest
import torch

import vpa
from tests import _loop_oracle as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def np64(t):
    return t.detach().double().cpu().numpy()


def problem(device, dtype, t, h, kvh, d, rot, *, sections=None, interleaved=False, far=5000,
            seed=0, norm=True, pos_dtype=torch.int64, theta=1e4):
    gen = torch.Generator().manual_seed(seed)
    qkv = torch.randn((t, (h + 2 * kvh) * d), generator=gen).to(dtype).to(device)
    q = qkv[:, :h * d].view(t, h, d)
    k = qkv[:, h * d:(h + kvh) * d].view(t, kvh, d)
    v = qkv[:, (h + kvh) * d:].view(t, kvh, d)
    inv_freq, axes = vpa.rotary_frequencies(rot, theta, device, sections=sections,
                                            interleaved=interleaved)
    n = 1 if sections is None else len(sections)
    pos = torch.randint(0, far, (n, t), generator=gen)
    pos = pos.to(torch.int32).view(torch.uint32) if pos_dtype == torch.uint32 else pos
    w = [(1 + 0.3 * torch.randn(d, generator=gen)).to(dtype).to(device) if norm else None
         for _ in range(2)]
    return q, k, v, pos.to(device), inv_freq, axes, w[0], w[1]


def check(got, x, pos, inv_freq, axes, w, adjacent=False, eps=1e-6):
    want, mag = ref.rotary(np64(x), pos.cpu().numpy(), inv_freq.cpu().numpy(),
                           None if axes is None else axes.cpu().numpy(),
                           weight=None if w is None else np64(w), eps=eps, adjacent=adjacent)
    info = torch.finfo(got.dtype)
    tol = np.abs(want) * info.eps / 2 + 24 * U * mag * (1 + info.eps) + info.smallest_normal * info.eps
    err = np.abs(np64(got) - want)
    assert np.all(err <= tol), (err - tol).max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 64), (96, 96), (192, 96), (256, 256), (128, 32),
                                   (16, 16), (80, 48), (240, 240)])
@pytest.mark.parametrize("adjacent", [False, True])
def test_rotary_qk_shapes(device, dtype, d, rot, adjacent):
    for t, h, kvh in [(1, 16, 8), (37, 3, 1), (130, 4, 4)]:
        q, k, _, pos, f, a, qw, kw = problem(device, dtype, t, h, kvh, d, rot, seed=t + d)
        oq, ok = vpa.rotary_qk(q, k, pos, f, a, q_norm=qw, k_norm=kw, adjacent=adjacent)
        check(oq, q, pos, f, a, qw, adjacent)
        check(ok, k, pos, f, a, kw, adjacent)


@pytest.mark.parametrize("sections,interleaved", [((24, 20, 20), False), ((24, 20, 20), True),
                                                  ((20, 30, 14), True), ((32, 32), True),
                                                  ((10, 20, 30, 4), False), ((64,), False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotary_axes(device, dtype, sections, interleaved):
    q, k, _, pos, f, a, qw, kw = problem(device, dtype, 65, 16, 8, 128, 128, sections=sections,
                                         interleaved=interleaved, seed=5)
    oq, ok = vpa.rotary_qk(q, k, pos, f, a, q_norm=qw, k_norm=kw)
    check(oq, q, pos, f, a, qw)
    check(ok, k, pos, f, a, kw)
    # an axis past the last counts as the last
    oq, _ = vpa.rotary_qk(q, k, pos[:1], f, a)
    check(oq, q, pos[:1], f, a, None)


def test_rotary_interleaved_axes_in_turn(device):
    _, a = vpa.rotary_frequencies(128, 1e6, device, sections=(24, 20, 20), interleaved=True)
    want = [i % 3 if i < 60 else 0 for i in range(64)]
    assert a.cpu().tolist() == want


@pytest.mark.parametrize("pos_dtype", [torch.int64, torch.uint32])
def test_rotary_far_positions_and_forms(device, pos_dtype):
    """Angles of a million turns and more keep their 64 bits; [T] positions, a
    view whose axes share one row, no axes, no norm on one side."""
    q, k, _, pos, f, a, qw, _ = problem(device, torch.float32, 50, 4, 2, 64, 64, far=2 ** 31 - 1,
                                        pos_dtype=pos_dtype, seed=9, theta=5e6)
    oq, ok = vpa.rotary_qk(q, k, pos[0], f, None, q_norm=qw)
    check(oq, q, pos, f, None, qw)
    check(ok, k, pos, f, None, None)
    _, axes = vpa.rotary_frequencies(64, 5e6, device, sections=(12, 10, 10))
    oq2, ok2 = vpa.rotary_qk(q, k, pos.expand(3, 50), f, axes, q_norm=qw)
    assert torch.equal(oq, oq2) and torch.equal(ok, ok2)


def test_rotary_negative_positions(device):
    q, k, _, pos, f, a, qw, kw = problem(device, torch.float32, 33, 2, 2, 64, 64, seed=3)
    oq, _ = vpa.rotary_qk(q, k, -pos, f, a)
    check(oq, q, -pos, f, a, None)


@pytest.mark.parametrize("dtype", TYPES)
def test_rotary_in_place_and_neighbours(device, dtype):
    """In place on slices of one projection: v and nothing else changes."""
    q, k, v, pos, f, a, qw, kw = problem(device, dtype, 41, 16, 8, 128, 64, seed=4)
    v0 = v.clone()
    want = vpa.rotary_qk(q, k, pos, f, a, q_norm=qw, k_norm=kw)
    got = vpa.rotary_qk(q, k, pos, f, a, q_norm=qw, k_norm=kw, out_q=q, out_k=k)
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(v, v0)


def test_rotary_zero_rows_zero_dims_zero_norm(device):
    q, k, _, pos, f, a, qw, kw = problem(device, torch.bfloat16, 4, 2, 2, 64, 64)
    oq, ok = vpa.rotary_qk(q[:0], k[:0], pos[:, :0], f, a)
    assert oq.shape == (0, 2, 64)
    empty = f[:0]
    oq, ok = vpa.rotary_qk(q, k, pos, empty, None)  # no rotated dims: a copy
    assert torch.equal(oq, q) and torch.equal(ok, k)
    z = torch.zeros_like(q)
    oq, _ = vpa.rotary_qk(z, k, pos, f, a, q_norm=qw, k_norm=kw)  # 0 / sqrt(eps)
    assert torch.equal(oq, z)


def make_caches(device, dtype, cache, nb, kvh, d, bs, seed):
    gen = torch.Generator().manual_seed(seed)
    if cache == "fp8":
        kc = torch.randint(0, 120, (nb, kvh, d // 16, bs, 16), generator=gen, dtype=torch.uint8)
        vc = torch.randint(0, 120, (nb, kvh, d, bs), generator=gen, dtype=torch.uint8)
        return kc.to(device), vc.to(device)
    x = 128 // torch.finfo(dtype).bits
    return (torch.randn((nb, kvh, d // x, bs, x), generator=gen).to(dtype).to(device),
            torch.randn((nb, kvh, d, bs), generator=gen).to(dtype).to(device))


def slots_for(rng, pattern, t, nb, bs):
    if pattern == "decode":  # one token in a block of its own, some padding
        s = rng.choice(nb, size=t, replace=False) * bs + rng.integers(0, bs, t)
        s[::5] = -1
        if t > 3:
            s[3] = nb * bs + 7  # past the pool
        return s
    start = rng.integers(0, bs)  # one run over whole blocks, from inside a block
    table = rng.permutation(nb)
    pos = start + np.arange(t)
    return table[pos // bs] * bs + pos % bs


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("d,bs", list(itertools.product([64, 96, 128, 192, 256], [8, 16, 32])))
def test_rotary_cache_is_both_ops(device, dtype, cache, d, bs):
    """q as rotary_qk gives it; over caches of the rows' type the keys and values are
    those of rotary_qk + reshape_and_cache bit for bit, untouched bytes among
    them. fp8 keys are rounded once from f32: within half a step of the exact
    value (2^-4 of it, 2^-10 below the normal range), and the two-step bytes'
    neighbours at most."""
    kvh, group, nb = 2, 3, 45
    rng = np.random.default_rng(d * bs)
    for pattern, t in [("decode", 1), ("decode", 19), ("run", 2 * bs + 5), ("run", 4 * bs)]:
        rot = d if t % 2 else d // 2 // 16 * 16
        q, k, v, pos, f, a, qw, kw = problem(device, dtype, t, kvh * group, kvh, d, rot, seed=t + d,
                                             norm=t != 19)
        kc, vc = make_caches(device, dtype, cache, nb, kvh, d, bs, seed=d + t)
        slots = slots_for(rng, pattern, t, nb, bs)
        sm = torch.from_numpy(slots.astype(np.int64)).to(device)
        ks = torch.tensor([0.013], device=device)
        vs = torch.tensor([0.02], device=device)
        kc2, vc2 = kc.clone(), vc.clone()
        oq, ok = vpa.rotary_qk(q, k, pos, f, a, q_norm=qw, k_norm=kw, adjacent=t == 19)
        vpa.reshape_and_cache(ok, v, ks, vs, kc2, vc2, sm)
        out = vpa.rotary_reshape_and_cache(q, k, v, pos, f, a, ks, vs, kc, vc, sm, q_norm=qw,
                                           k_norm=kw, adjacent=t == 19)
        assert torch.equal(out, oq)
        assert torch.equal(vc, vc2)
        if cache == "same":
            assert torch.equal(kc, kc2)
            continue
        live = (slots >= 0) & (slots < nb * bs)
        want, mag = ref.rotary(np64(k), pos.cpu().numpy(), f.cpu().numpy(), a.cpu().numpy(),
                               weight=None if kw is None else np64(kw), adjacent=t == 19)
        keys = kc.view(torch.float8_e4m3fn).float().cpu().numpy().astype(np.float64)
        got = keys.transpose(0, 3, 1, 2, 4).reshape(nb * bs, kvh, d)[slots[live]]
        exact = np.clip(want[live] / 0.013, -448, 448)
        tol = np.maximum(np.abs(exact) * 2.0 ** -4, 2.0 ** -10) + 30 * U * mag[live] / 0.013
        assert np.all(np.abs(got - exact) <= tol)
        # everything else is as it was
        rest = np.setdiff1d(np.arange(nb * bs), slots[live])
        a8 = kc.cpu().numpy().transpose(0, 3, 1, 2, 4).reshape(nb * bs, kvh, d)
        b8 = kc2.cpu().numpy().transpose(0, 3, 1, 2, 4).reshape(nb * bs, kvh, d)
        assert np.array_equal(a8[rest], b8[rest])


def test_rotary_cache_strided_pool_and_in_place(device):
    """Caches that are views into a larger pool (padded head strides); out = q."""
    t, kvh, d, bs, nb = 21, 4, 128, 16, 9
    q, k, v, pos, f, a, qw, kw = problem(device, torch.bfloat16, t, 8, kvh, d, d, seed=8)
    pool_k = torch.zeros((nb, kvh + 2, d // 8, bs, 8), dtype=torch.bfloat16, device=device)
    pool_v = torch.zeros((nb, kvh + 2, d, bs), dtype=torch.bfloat16, device=device)
    kc, vc = pool_k[:, 1:1 + kvh], pool_v[:, 1:1 + kvh]
    kc2, vc2 = kc.contiguous().clone(), vc.contiguous().clone()
    sm = torch.arange(5, 5 + t, device=device)
    want = vpa.rotary_reshape_and_cache(q, k, v, pos, f, a, None, None, kc2, vc2, sm, q_norm=qw,
                                        k_norm=kw)
    got = vpa.rotary_reshape_and_cache(q, k, v, pos, f, a, None, None, kc, vc, sm, q_norm=qw,
                                       k_norm=kw, out=q)
    assert got is q and torch.equal(got, want)
    assert torch.equal(kc, kc2) and torch.equal(vc, vc2)
    assert not pool_k[:, 0].any() and not pool_k[:, -1].any() and not pool_v[:, 0].any()


def test_rotary_in_a_graph(device):
    q, k, v, pos, f, a, qw, kw = problem(device, torch.bfloat16, 17, 16, 8, 128, 128, seed=2,
                                         sections=(24, 20, 20))
    kc, vc = make_caches(device, torch.bfloat16, "same", 40, 8, 128, 16, 1)
    sm = torch.arange(0, 17 * 16, 16, device=device)
    oq, ok = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty_like(
        k, memory_format=torch.contiguous_format)
    out = torch.empty_like(oq)

    def step():
        vpa.rotary_qk(q, k, pos, f, a, q_norm=qw, k_norm=kw, out_q=oq, out_k=ok)
        vpa.rotary_reshape_and_cache(q, k, v, pos, f, a, None, None, kc, vc, sm, q_norm=qw,
                                     k_norm=kw, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        pos.add_(37 * i + 1)
        q.normal_()
        sm.add_(1)
        graph.replay()
        got = [x.clone() for x in (oq, ok, out, kc, vc)]
        torch.cuda.synchronize()
        kc.zero_()
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got[:3] + got[4:], (oq, ok, out, vc)))
        blk = sm // 16
        assert torch.equal(got[3][blk, :, :, sm % 16], kc[blk, :, :, sm % 16])
