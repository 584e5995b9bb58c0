"""GPU tests of the block-scaled cache: the append bit for bit (bytes and scales), the
attention within the bound that its roundings add up to (``attention_bound``)."""

import numpy as np
import pytest
import torch

import vpa
from tests import _serving_oracle as ref
from tests._util import block_tables_for, i64, u32

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = list(UNIT)
NAN_BYTES = (0x7F, 0xFF)


def pool(rng, nb, kvh, d, bs, spread=3):
    """Bytes and power-of-two scales of a pool: any finite bytes, uneven blocks."""
    out = []
    for shape in ((nb, kvh, d // 16, bs, 16), (nb, kvh, d, bs)):
        b = ref.e4m3((rng.standard_normal(shape) * 60).astype(np.float32))
        out += [b, 2.0 ** rng.integers(-8, -8 + spread, size=(nb, kvh)).astype(np.float64)]
    return out  # kc, ks, vc, vs


def dev(a, device, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(device)
    return t if dtype is None else t.to(dtype)


def rows_of(rng, t, kvh, d, dtype, device, wide=0):
    x = (rng.standard_normal((t, kvh, d + wide)) * 2.0 ** rng.integers(-3, 4, size=(t, 1, 1)))
    x = torch.from_numpy(x.astype(np.float32)).to(dtype)[..., :d]
    return x.to(device)


def check_append(device, key, value, state, slots):
    kc, ks, vc, vs = (a.copy() for a in state)
    got = [dev(kc, device), dev(ks, device, torch.float32), dev(vc, device),
           dev(vs, device, torch.float32)]
    vpa.reshape_and_cache_block_scaled(key, value, got[1], got[3], got[0], got[2], i64(slots, device))
    torch.cuda.synchronize()
    ref.append(key.float().cpu().numpy(), value.float().cpu().numpy(), ks, vs, kc, vc, slots)
    for name, g, w in zip(("key scales", "value scales"), (got[1], got[3]), (ks, vs)):
        assert np.array_equal(g.cpu().numpy().astype(np.float64), w), name
    for name, g, w in zip(("key cache", "value cache"), (got[0], got[2]), (kc, vc)):
        g = g.cpu().numpy()
        nan = (w & 127) == 127
        assert np.array_equal((g & 127) == 127, nan), name
        assert np.array_equal(g[~nan], w[~nan]), (name, np.argwhere((g != w) & ~nan)[:5])
    return got


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d,bs", [(64, 8), (64, 32), (96, 16), (128, 8), (128, 16), (192, 32),
                                  (256, 8), (256, 32)])
def test_append_bits(device, dtype, d, bs):
    rng = np.random.default_rng(d + bs)
    kvh, nb = 3, 40
    state = pool(rng, nb, kvh, d, bs)
    blocks = rng.permutation(np.arange(1, nb))
    slots = []
    # whole blocks, a block's end and the next one's start, single tokens, padding
    slots += list(blocks[0] * bs + np.arange(bs))
    slots += [-1, -5]
    slots += list(blocks[1] * bs + np.arange(3, bs)) + list(blocks[2] * bs + np.arange(2))
    slots += [nb * bs, nb * bs + 7]
    slots += [int(b) * bs + int(rng.integers(bs)) for b in blocks[3:14]]
    key = rows_of(rng, len(slots), kvh, d, dtype, device)
    value = rows_of(rng, len(slots), kvh, d, dtype, device)
    check_append(device, key, value, state, np.array(slots))


@pytest.mark.parametrize("dtype,d,bs", [(torch.bfloat16, 128, 16), (torch.float32, 64, 8),
                                        (torch.float16, 96, 32)])
def test_append_many_tokens(device, dtype, d, bs):
    """From 2048 tokens on a workgroup looks through a block's worth of them."""
    rng = np.random.default_rng(7)
    kvh, run = 2, 5 * bs + 3
    n = 2048 // run + 2
    need = n * (run // bs + 2)
    nb = need + 3
    blocks = rng.permutation(np.arange(1, nb))
    slots = []
    for i in range(n):
        start = int(rng.integers(bs))
        mine = blocks[i * (run // bs + 2):(i + 1) * (run // bs + 2)]
        slots += [int(mine[(start + t) // bs]) * bs + (start + t) % bs for t in range(run)]
        slots += [-1] * int(rng.integers(3))
    assert len(slots) >= 2048
    state = pool(rng, nb, kvh, d, bs)
    key = rows_of(rng, len(slots), kvh, d, dtype, device)
    value = rows_of(rng, len(slots), kvh, d, dtype, device)
    check_append(device, key, value, state, np.array(slots))


def test_append_special_values(device):
    """Zeros, infinities, NaN, numbers at E4M3's and the types' ends, unset scales."""
    rng = np.random.default_rng(3)
    kvh, d, bs, nb = 1, 64, 16, 12
    kc, ks, vc, vs = pool(rng, nb, kvh, d, bs)
    kc[3, 0, 0, 0, :2] = NAN_BYTES
    ks[4], vs[4] = 0.0, 0.0
    rows = np.zeros((10, kvh, d), np.float32)
    rows[0] = 0.0                                       # block 1, opened by zeros
    rows[1, 0, :3] = [np.inf, -np.inf, 3.0]             # block 2, opened
    rows[2, 0, :2] = [np.nan, 1000.0]                   # block 3, NaN in it already
    rows[3, 0, 0] = 1e-3                                # block 4: unset scale, inside
    rows[4, 0, :3] = [448.0, 224.0, 449.0]              # block 5
    rows[5, 0, 0] = 448.0                               # block 6: s = 1
    rows[6, 0, 0] = np.nextafter(np.float32(448.0), np.float32(500))  # block 7: s = 2
    rows[7, 0, :2] = [3.3e38, -1.0]                     # block 8
    rows[8, 0, :2] = [1e-40, 2.0 ** -126]               # block 9: below the least scale
    rows[9, 0] = np.nan                                 # block 10: nothing finite
    slots = np.array([1 * bs, 2 * bs, 3 * bs + 5, 4 * bs + 1, 5 * bs, 6 * bs, 7 * bs, 8 * bs, 9 * bs,
                      10 * bs])
    x = torch.from_numpy(rows).to(device)
    got = check_append(device, x, x.clone(), (kc, ks, vc, vs), slots)
    scales = got[1].cpu().numpy()[:, 0]
    assert scales[1] == 2.0 ** -100 and scales[6] == 1.0 and scales[7] == 2.0
    assert scales[9] == 2.0 ** -100 and scales[10] == 2.0 ** -100


def test_append_token_by_token_grows_the_scale(device):
    """A decode's tokens, each louder than the one before: every step bit for bit, and the
    block still holds each token within E4M3's half step of it (powers of two lose
    nothing until a value leaves E4M3's normal range)."""
    rng = np.random.default_rng(5)
    kvh, d, bs, nb = 2, 128, 16, 3
    kc, ks, vc, vs = pool(rng, nb, kvh, d, bs)
    rows = []
    for t in range(bs):
        x = rng.uniform(0.5, 1.0, (1, kvh, d)).astype(np.float32) * np.float32(1.3 ** t)
        rows.append(x)
        x = torch.from_numpy(x).to(device)
        got = check_append(device, x, x.clone(), (kc, ks, vc, vs), np.array([2 * bs + t]))
        kc, vc = got[0].cpu().numpy(), got[2].cpu().numpy()
        ks, vs = (got[i].cpu().numpy().astype(np.float64) for i in (1, 3))
    back = ref.e4m3_value(vc[2]) * vs[2][:, None, None]
    want = np.concatenate(rows).transpose(1, 2, 0)
    assert np.all(np.abs(back - want) <= 2.0 ** -4 * want)


def test_append_repeated_slots_and_strides(device):
    """Pad rows that all name slot 0: the last counts. Rows that are slices of a
    projection, scales and caches that are slices of larger pools."""
    rng = np.random.default_rng(9)
    kvh, d, bs, nb = 2, 64, 16, 6
    state = pool(rng, nb, kvh, d, bs)
    slots = np.array([3 * bs + 2] + [0] * 70)
    packed = rows_of(rng, len(slots), 2 * kvh, d, torch.bfloat16, device)
    key, value = packed[:, :kvh], packed[:, kvh:]
    check_append(device, key, value, state, slots)
    # views
    kc, ks, vc, vs = (a.copy() for a in state)
    big = [torch.zeros((nb, kvh + 2) + a.shape[2:], dtype=torch.uint8, device=device) for a in (kc, vc)]
    scl = [torch.zeros((nb, kvh + 5), device=device) for _ in range(2)]
    for b, a in zip(big, (kc, vc)):
        b[:, 1:1 + kvh] = dev(a, device)
    for b, a in zip(scl, (ks, vs)):
        b[:, 3:3 + kvh] = dev(a, device, torch.float32)
    vpa.reshape_and_cache_block_scaled(key, value, scl[0][:, 3:3 + kvh], scl[1][:, 3:3 + kvh],
                                       big[0][:, 1:1 + kvh], big[1][:, 1:1 + kvh], i64(slots, device))
    torch.cuda.synchronize()
    ref.append(key.float().cpu().numpy(), value.float().cpu().numpy(), ks, vs, kc, vc, slots)
    for b, a in zip(big, (kc, vc)):
        assert np.array_equal(b[:, 1:1 + kvh].cpu().numpy(), a)
        assert not b[:, 0].any() and not b[:, 1 + kvh:].any()
    for b, a in zip(scl, (ks, vs)):
        assert np.array_equal(b[:, 3:3 + kvh].cpu().numpy().astype(np.float64), a)
        assert not b[:, :3].any() and not b[:, 3 + kvh:].any()


# ---- attention ----------------------------------------------------------------


class Problem:
    def __init__(self, device, seed, dtype, heads, kvh, d, bs, lens, rows=None, pad_cols=0,
                 any_scale=False, spread=3):
        rng = np.random.default_rng(seed)
        self.device, self.dtype, self.lens = device, dtype, np.asarray(lens)
        nb = int((-(-self.lens // bs)).sum()) + 4
        self.kc, self.ks, self.vc, self.vs = pool(rng, nb, kvh, d, bs, spread)
        if any_scale:
            self.ks *= rng.uniform(0.5, 1.0, self.ks.shape)
            self.vs *= rng.uniform(0.5, 1.0, self.vs.shape)
        self.ks, self.vs = self.ks.astype(np.float32), self.vs.astype(np.float32)
        self.tables = block_tables_for(rng, list(self.lens), nb, bs, pad_cols=pad_cols)
        self.cu = None
        total = len(self.lens)
        if rows is not None:
            self.cu = np.concatenate([[0], np.cumsum(rows)])
            total = int(self.cu[-1])
        q = rng.standard_normal((total, heads, d)).astype(np.float32)
        self.q = torch.from_numpy(q).to(dtype)
        self.scale, self.bs = d ** -0.5, bs
        # what stands behind a context is nobody's: NaN
        for s, size in enumerate(self.lens):
            if size % bs:
                b = self.tables[s, size // bs]
                self.kc[b][:, :, size % bs:] = 0x7F
                self.vc[b][:, :, size % bs:] = 0xFF

    def run(self, causal=True, max_len=None, **kw):
        cu = None if self.cu is None else u32(self.cu, self.device)
        out = vpa.paged_attention_block_scaled(
            self.q.to(self.device), dev(self.ks, self.device), dev(self.vs, self.device),
            dev(self.kc, self.device), dev(self.vc, self.device), u32(self.tables, self.device),
            u32(self.lens, self.device), self.scale, cu_seqlens_q=cu, causal=causal,
            max_context_len=max_len, **kw)
        torch.cuda.synchronize()
        return out

    def check(self, causal=True, **kw):
        got = self.run(causal, **kw).float().cpu().numpy().astype(np.float64)
        eps = kw.get("denom_eps")
        eps = (0.0 if causal and self.cu is not None else 1e-6) if eps is None else eps
        want, *rest = ref.attention(self.q.float().numpy(), self.ks, self.vs, self.kc, self.vc,
                                    self.tables, self.lens, self.scale, self.cu, causal, eps)
        bound = ref.attention_bound(want, *rest, self.q.shape[2], int(self.lens.max(initial=1)),
                                    UNIT[self.dtype])
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(got), nan)
        worst = np.max((np.abs(got - want) / bound)[~nan], initial=0.0)
        assert worst <= 1.0, worst
        return got


SHAPES = [(d, bs) for d in (64, 96, 128, 192, 256) for bs in (8, 16, 32)]


@pytest.mark.parametrize("d,bs", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_decode(device, dtype, d, bs):
    Problem(device, d * bs, dtype, 6, 2, d, bs, [1, 700, 33, 0, 64, 257], any_scale=True).check()


@pytest.mark.parametrize("d,bs", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_prompt_rows(device, dtype, d, bs):
    p = Problem(device, d + bs, dtype, 4, 2, d, bs, [90, 37, 130], rows=[41, 37, 5], pad_cols=3)
    p.check()


@pytest.mark.parametrize("heads,kvh", [(1, 1), (8, 8), (14, 2), (16, 1), (17, 1), (40, 2), (64, 1),
                                       (130, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_groups(device, dtype, heads, kvh):
    Problem(device, heads, dtype, heads, kvh, 64, 16, [100, 1, 333], any_scale=True).check()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows", [[8, 1, 3], [70, 130, 1], [20, 16, 17], [200, 0, 64]])
def test_rows_and_masks(device, dtype, rows, causal):
    Problem(device, sum(rows), dtype, 4, 2, 128, 16, [300, 140, 70], rows=rows).check(causal)


@pytest.mark.parametrize("lens,rows", [([5000], None), ([2304, 2305, 1, 0], None),
                                       ([3000, 260], [20, 20]), ([1800], [100]), ([4096], [3])])
def test_keys_split_over_workgroups(device, lens, rows):
    for dtype in (torch.bfloat16, torch.float32):
        Problem(device, 4, dtype, 4, 2, 64, 16, lens, rows=rows).check()


def test_batches_of_many_short_contexts(device):
    rng = np.random.default_rng(0)
    Problem(device, 1, torch.bfloat16, 4, 2, 64, 16, rng.integers(0, 90, size=300)).check()


@pytest.mark.parametrize("dtype,batch,hi,rows,causal", [
    (torch.bfloat16, 700, 64, 0, True), (torch.float32, 700, 120, 0, True),
    (torch.float16, 40, 500, 110, True), (torch.float32, 60, 64, 70, False),
    (torch.bfloat16, 200, 130, 25, False)])
def test_batches_whose_waves_have_rows_of_their_own(device, dtype, batch, hi, rows, causal):
    """Short contexts of many sequences, whose keys are not split."""
    rng = np.random.default_rng(batch)
    lens = rng.integers(0, hi + 1, size=batch)
    lens[0] = hi
    n = None if rows == 0 else rng.integers(0, rows + 1, size=batch)
    Problem(device, 5, dtype, 4, 2, 64, 16, lens, rows=n, any_scale=True).check(causal)


def test_more_rows_than_tokens(device):
    """The first rows see nothing and are zeros."""
    p = Problem(device, 2, torch.bfloat16, 4, 2, 64, 16, [5, 0, 20], rows=[12, 3, 20])
    got = p.check()
    assert not got[:7].any() and not got[12:15].any()
    assert got[7:12].any()


@pytest.mark.parametrize("rows", [None, [30, 9, 40]])
def test_absent_blocks_and_stale_bytes(device, rows):
    """Ids past the pool (their tokens are left out), one of a whole context, and a table
    wider than the contexts whose other entries are such ids."""
    p = Problem(device, 3, torch.float16, 4, 2, 128, 16, [200, 9, 64], rows=rows, pad_cols=5)
    p.tables[0, 3] = p.tables[2, 0] = 5000
    p.tables[1, 0] = 0xFFFFFFFF
    for s, size in enumerate(p.lens):
        p.tables[s, -(-size // 16):] = 0xFFFFFFFF
    got = p.check()
    lone = slice(1, 2) if rows is None else slice(30, 39)
    assert not got[lone].any()


@pytest.mark.parametrize("rows", [[40], [150]])
def test_nan_of_a_later_token_stays_there(device, rows):
    """A NaN in V (or K) of a token reaches the rows that see it and no others."""
    p = Problem(device, 6, torch.bfloat16, 2, 1, 64, 16, [200], rows=rows)
    n, size = rows[0], 200
    late = size - 7
    p.vc[p.tables[0, late // 16], 0, 5, late % 16] = 0x7F
    got = p.check()
    assert np.isnan(got[n - 7:, :, 5]).all() and not np.isnan(got[:n - 7]).any()
    assert not np.isnan(np.delete(got, 5, axis=2)).any()
    p.kc[p.tables[0, late // 16], 0, 0, late % 16, 3] = 0xFF
    got = p.check()
    assert np.isnan(got[n - 7:]).all() and not np.isnan(got[:n - 7]).any()


@pytest.mark.parametrize("rows", [None, [40, 3], [300, 2]])
@pytest.mark.parametrize("size", [60, 900, 6000])
def test_nan_queries_and_keys(device, rows, size):
    """NaN wherever a row's query, or a key that it sees, holds one: also where every key of
    a wave's or of a chunk's is such."""
    p = Problem(device, 16, torch.bfloat16, 2, 1, 64, 16, [size, 100], rows=rows)
    p.q[0, 1, 7] = float("nan")
    got = p.check()
    seen = rows is None or size >= rows[0]
    assert np.isnan(got[0, 1]).all() == seen and not np.isnan(got[0, 0]).any()
    p.kc[p.tables[1, :4], :, 1, :, 3] = 0x7F
    got = p.check()
    assert np.isnan(got[-1]).all()


def test_scales_far_apart(device):
    """Blocks whose values differ by 2^40: the small ones vanish in the sum, nothing else
    does; values and scales that f16 cannot hold."""
    for shift in (0, 60, -60):
        p = Problem(device, 8, torch.float16, 4, 2, 64, 8, [150, 40], spread=20)
        p.vs = np.ldexp(p.vs, shift).astype(np.float32)
        p.ks[:] = 2.0 ** -7
        for dtype in (torch.bfloat16, torch.float32):
            p.dtype, p.q = dtype, p.q.to(dtype)
            p.check()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 0.3])
@pytest.mark.parametrize("rows", [None, [300, 20]])
def test_any_softmax_scale(device, dtype, scale, rows):
    """Negative, zero and tiny softmax scales, over scales of 1 and of other sizes, in contexts
    of many steps."""
    for ks in (None, 1.0, 2.0 ** -3):
        p = Problem(device, 9, dtype, 4, 2, 64, 16, [1500, 700], rows=rows)
        p.scale = scale
        if ks is not None:
            p.ks[:] = ks
            p.ks[p.tables[0, 40:]] = 2.0 ** -7
        p.q = (p.q.float() / 64).to(dtype)
        p.check()


def test_scales_that_turn_odd(device):
    """Powers of two, then others, then smaller ones, absent blocks among them."""
    for rows in (None, [250, 40]):
        p = Problem(device, 19, torch.bfloat16, 4, 2, 64, 8, [1300, 600], rows=rows)
        cols = p.tables.shape[1]
        for s in (p.ks, p.vs):
            s[p.tables[0, 30:60]] *= 0.7
            s[p.tables[0, 90:95]] *= 2.0 ** -12
            s[p.tables[0, 100:]] *= 2.0 ** -4
            s[p.tables[1, 10]] = 0.0
        p.tables[0, 70] = 0xFFFFFFFF
        assert cols > 100
        p.check()


def test_zero_scales_and_negative_softmax_scale(device):
    p = Problem(device, 9, torch.bfloat16, 4, 2, 64, 16, [100, 50])
    p.scale = -0.2
    p.check()
    p.vs[:] = 0.0
    p.ks[p.tables[0, 1]] = 0.0
    assert not p.check().any()


def test_limits_given_by_the_caller(device):
    """max_context_len and max_query_len clamp, rows past total_query_rows are left."""
    p = Problem(device, 10, torch.bfloat16, 4, 2, 64, 16, [90, 60], rows=[10, 6])
    want = p.run().clone()
    assert torch.equal(p.run(max_len=96), want)
    short = Problem(device, 10, torch.bfloat16, 4, 2, 64, 16, [90, 60], rows=[10, 6])
    short.lens = np.minimum(short.lens, 40)
    assert torch.equal(p.run(max_len=40), short.run(max_len=40))
    # more rows promised by cu_seqlens_q than there are
    q = p.q[:12].to(device)
    out = torch.full((14, 4, 64), 7.0, dtype=torch.bfloat16, device=device)
    vpa.paged_attention_block_scaled(
        q, dev(p.ks, device), dev(p.vs, device), dev(p.kc, device), dev(p.vc, device),
        u32(p.tables, device), u32(p.lens, device), p.scale, cu_seqlens_q=u32(p.cu, device),
        max_query_len=10, max_context_len=90, out=out[:12])
    assert torch.equal(out[:10], want[:10]) and bool((out[12:] == 7).all())


def test_results_do_not_vary(device):
    p = Problem(device, 11, torch.bfloat16, 8, 2, 128, 16, [3000, 1200, 77], rows=[30, 8, 70])
    first = p.run().clone()
    for _ in range(3):
        assert torch.equal(p.run().view(torch.int16), first.view(torch.int16))


def test_own_workspace_and_out(device):
    p = Problem(device, 12, torch.bfloat16, 8, 2, 64, 16, [3000, 10])
    ws = vpa.paged_attention_block_scaled_workspace(2, 8, 2, 64, 3000, torch.bfloat16, device)
    assert ws is not None
    out = torch.empty((2, 8, 64), dtype=torch.bfloat16, device=device)
    want = p.run()
    assert p.run(out=out, workspace=ws) is out and torch.equal(out, want)
    with pytest.raises(vpa.VpaError, match="bytes needed"):
        p.run(workspace=ws[:-256])


def test_far_blocks(device):
    """A pool of more than 4 GiB: blocks whose offsets pass 32 bits."""
    nb, kvh, d, bs = 560000, 1, 256, 32
    kc = torch.zeros((nb, kvh, d // 16, bs, 16), dtype=torch.uint8, device=device)
    vc = torch.zeros((nb, kvh, d, bs), dtype=torch.uint8, device=device)
    assert kc.numel() > 1 << 32
    ks, vs = vpa.block_scales(nb, kvh, device)
    rng = np.random.default_rng(1)
    k, v = rows_of(rng, 40, kvh, d, torch.bfloat16, device), rows_of(rng, 40, kvh, d, torch.bfloat16, device)
    far = nb - 1
    slots = np.concatenate([far * bs + np.arange(bs), (far - 2) * bs + np.arange(40 - bs)])
    vpa.reshape_and_cache_block_scaled(k, v, ks, vs, kc, vc, i64(slots, device))
    small = [np.zeros((3,) + tuple(t.shape[1:]), np.uint8) for t in (kc, vc)]
    sk, sv = np.zeros((3, kvh)), np.zeros((3, kvh))
    at = np.concatenate([1 * bs + np.arange(bs), 2 * bs + np.arange(40 - bs)])
    ref.append(k.float().cpu().numpy(), v.float().cpu().numpy(), sk, sv, small[0], small[1], at)
    for i, b in ((1, far), (2, far - 2)):
        assert np.array_equal(kc[b].cpu().numpy(), small[0][i]) and np.array_equal(vc[b].cpu().numpy(), small[1][i])
    q = torch.from_numpy(rng.standard_normal((1, 2, d)).astype(np.float32)).to(device)
    got = vpa.paged_attention_block_scaled(q, ks, vs, kc, vc, u32([[far, far - 2]], device),
                                           u32([40], device), d ** -0.5, max_context_len=40)
    want, *rest = ref.attention(q.cpu().numpy(), sk, sv, small[0], small[1], np.array([[1, 2]]), [40],
                                d ** -0.5, eps=1e-6)
    assert np.all(np.abs(got.cpu().numpy() - want) <= ref.attention_bound(want, *rest, d, 40, 2.0 ** -24))
