"""The decode loop's operators run together, as a server uses them, against a host
model in 64 bits: prompts rotated into the cache, their window's attention weights,
the cache cut by them and its blocks given back, a decode step that goes on from there,
drafted tokens verified and the rejected ones taken back, one more step.

The host model knows each sequence as a list of its original tokens per kv head, and
what each token's exact key and value are. Keys in the cache are f32: within one
rounding (2^-24 of the value) and the rotation's own 30 * 2^-24 of |x_a| + |x_b|, the
bound of the rotary tests. Attention over f32 caches is held to the framework's 1e-5.
A token's weight is off by the bound that the tests of the weights derive."""

import numpy as np
import pytest
import torch

import vpa
from tests import _loop_oracle as ref
from tests._util import assert_attention_close, u32
from oracle import oracle as orc

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
H, KVH, D, BS, COLS, NB = 6, 2, 64, 16, 12, 60
SCALE = D ** -0.5
SECTIONS = (16, 8, 8)


def np64(t):
    return t.detach().double().cpu().numpy()


class Loop:
    def __init__(self, device):
        self.device = device
        self.gen = torch.Generator().manual_seed(3)
        self.alloc = vpa.DeviceBlockAllocator(NB, BS, 3, COLS, device)
        self.kc = torch.full((NB, KVH, D // 4, BS, 4), float("nan"), device=device)
        self.vc = torch.full((NB, KVH, D, BS), float("nan"), device=device)
        self.inv_freq, self.axes = vpa.rotary_frequencies(D, 1e6, device, sections=SECTIONS,
                                                          interleaved=True)
        self.scores = torch.zeros((3, KVH, COLS * BS), device=device)
        self.want_scores = np.zeros((3, KVH, COLS * BS))
        self.tokens = [[[] for _ in range(KVH)] for _ in range(3)]  # (key, key's bound, value)
        self.next_pos = [0, 0, 0]  # rotary positions go on whatever is cut

    def tables(self):
        return self.alloc.block_tables.cpu().numpy().view(np.uint32)

    def append(self, rows, slots):
        """New rows for every sequence through the fused append; returns the rotated q."""
        n = sum(rows)
        q, k, v = (torch.randn((n, h, D), generator=self.gen).to(self.device) for h in (H, KVH, KVH))
        first = np.concatenate([p + np.arange(r) for p, r in zip(self.next_pos, rows)])
        pos = np.stack([first, first // 3, first % 7])
        got_q = vpa.rotary_reshape_and_cache(
            q, k, v, torch.from_numpy(pos).to(self.device), self.inv_freq, self.axes, None, None,
            self.kc, self.vc, slots)
        args = (pos, np64(self.inv_freq), self.axes.cpu().numpy())
        want_q, mag_q = ref.rotary(np64(q), *args)
        assert np.all(np.abs(np64(got_q) - want_q) <= U * np.abs(want_q) + 30 * U * mag_q)
        keys, mag = ref.rotary(np64(k), *args)
        bound, i = U * np.abs(keys) + 30 * U * mag, 0
        for s, r in enumerate(rows):
            for t in range(i, i + r):
                for j in range(KVH):
                    self.tokens[s][j].append((keys[t, j], bound[t, j], np64(v)[t, j]))
            i += r
            self.next_pos[s] += r
        return got_q

    def check_cache(self):
        """Each sequence's cache holds its tokens; returns its exact reading."""
        kc, vc, tables = np64(self.kc), np64(self.vc), self.tables()
        for s in range(3):
            n = len(self.tokens[s][0])
            k, v = ref.rows_of(kc, tables[s], n), ref.rows_of(vc, tables[s], n)
            for j in range(KVH):
                want = [np.stack(x) for x in zip(*self.tokens[s][j])]
                assert np.all(np.abs(k[j] - want[0]) <= want[1])
                assert np.array_equal(v[j], want[2])
        return kc, vc, tables

    def check_attention(self, got, q, rows, causal=True):
        kc, vc, tables = self.check_cache()
        q, want, i = np64(q), [], 0
        for s, r in enumerate(rows):
            n = len(self.tokens[s][0])
            k, v = ref.rows_of(kc, tables[s], n), ref.rows_of(vc, tables[s], n)
            for t in range(r):
                see = n - r + t + 1 if causal else n
                for h in range(H):
                    j = h // (H // KVH)
                    p = ref.softmax(SCALE * (k[j, :see] @ q[i + t, h]), 1.0)
                    want.append(p @ v[j, :see])
            i += r
        assert_attention_close(got.float().cpu().numpy().reshape(-1, D), np.stack(want), orc.F32)

    def check_weights(self, q, rows, lens):
        cu = np.concatenate([[0], np.cumsum(rows)])
        kc, _, tables = self.check_cache()
        before = self.want_scores
        want = ref.attention_weights(np64(q), kc, tables, lens, SCALE, before, cu, True)
        size = SCALE * np.abs(np64(q)).sum(-1).max() * np.nanmax(np.abs(kc))
        rel = 2 * (D + 3) * U * size + (24 + 2 * size) * U
        tol = (want - before) * rel + want * (max(rows) * H // KVH + 2) * U
        assert np.all(np.abs(np64(self.scores) - want) <= tol)
        self.want_scores = np64(self.scores)  # goes on from what the device holds


def test_loop(device):
    m = Loop(device)
    alloc = m.alloc

    # prompts of ragged length, straight into the cache
    lens = [50, 23, 130]
    assert alloc.allocate(u32(lens, device)).all()
    slots = np.concatenate([m.tables()[s, np.arange(n) // BS].astype(np.int64) * BS + np.arange(n) % BS
                            for s, n in enumerate(lens)])
    q = m.append(lens, torch.from_numpy(slots).to(device))
    cu = u32(np.concatenate([[0], np.cumsum(lens)]), device)
    out = vpa.paged_attention_varlen_prefill(q, m.kc, m.vc, alloc.block_tables, u32(lens, device), cu,
                                             None, None, SCALE, 1.0, causal=True)
    m.check_attention(out, q, lens)

    # the weights of the last rows of each prompt
    window = [8, 8, 8]
    ends = np.cumsum(lens)
    qw = torch.cat([q[e - 8:e] for e in ends])
    vpa.paged_attention_weights(qw, m.kc, None, alloc.block_tables, u32(lens, device), SCALE, m.scores,
                                cu_seqlens_q=u32([0, 8, 16, 24], device), max_query_len=8)
    m.check_weights(qw, window, lens)

    # cut to 40 tokens; the blocks behind go back
    free = int(alloc.free_ring_state[1])
    old_lens, kept = ref.evict(np64(m.scores), lens, 40, 2, 8)
    new_lens, got_kept = vpa.evict_kv_cache(m.kc, m.vc, m.scores, alloc.block_tables,
                                            u32(lens, device), 40, keep_first=2, keep_last=8)
    assert new_lens.cpu().numpy().tolist() == old_lens.tolist() == [40, 23, 40]
    for s in range(3):
        for j in range(KVH):
            ids = kept[s][j]
            assert got_kept[s, j, :len(ids)].cpu().numpy().tolist() == ids.tolist()
            m.tokens[s][j] = [m.tokens[s][j][t] for t in ids]
            row = np.zeros(COLS * BS)
            row[:len(ids)] = m.want_scores[s, j, ids]
            m.want_scores[s, j] = row
    assert np.array_equal(np64(m.scores), m.want_scores)
    alloc.trim(new_lens)
    assert alloc.row_blocks.cpu().numpy().tolist() == [3, 2, 3]
    assert int(alloc.free_ring_state[1]) == free + (4 - 3) + (9 - 3)
    m.check_cache()

    # a decode step goes on behind what is left
    slots, ctx = alloc.step()
    assert ctx.cpu().numpy().tolist() == [41, 24, 41]
    q = m.append([1, 1, 1], slots)
    out = vpa.paged_attention(q, None, None, m.kc, m.vc, alloc.block_tables, ctx, None, 41, SCALE, 1.0,
                              None)
    m.check_attention(out, q, [1, 1, 1])
    vpa.paged_attention_weights(q, m.kc, None, alloc.block_tables, ctx, SCALE, m.scores)
    m.check_weights(q, [1, 1, 1], [41, 24, 41])

    # the step's token and three drafts behind it, verified at once
    held = np.array([41, 24, 41])
    rows = [4, 4, 4]
    assert alloc.allocate(u32(held + 4, device)).all()
    at = held[:, None] + np.arange(4)
    slots = np.take_along_axis(m.tables().astype(np.int64), at // BS, 1) * BS + at % BS
    q = m.append(rows, torch.from_numpy(slots.reshape(-1)).to(device))
    out = vpa.paged_attention_varlen_prefill(q, m.kc, m.vc, alloc.block_tables, u32(held + 4, device),
                                             u32([0, 4, 8, 12], device), None, None, SCALE, 1.0,
                                             causal=True)
    m.check_attention(out, q, rows)
    target = torch.randn((3, 4, 700), generator=m.gen) * 3
    draft = target[:, :3] + torch.randn((3, 3, 700), generator=m.gen)
    draft[0, 0, target[0, 0].argmin()] = 20.0  # the drafter is sure of it: refused
    ids = draft.argmax(-1).to(torch.int32)
    accept, sample = torch.full((3, 3), 0.4), torch.tensor([0.1, 0.5, 0.9])
    accept[1] = 0.0  # and these are all taken
    want_ids, want_count, margin = ref.verify(target.numpy(), ids.numpy(), accept.numpy(),
                                              sample.numpy(), draft.numpy())
    assert margin.min() > 1e-9 and want_count[0] == 1 and want_count[1] == 4
    got_ids, count = vpa.verify_draft_tokens(
        target.to(device), u32(ids.numpy(), device), accept.to(device), sample.to(device),
        draft_logits=draft.to(device))
    assert np.array_equal(got_ids.cpu().numpy(), want_ids)
    assert np.array_equal(count.cpu().numpy(), want_count)

    # the step's token and the accepted drafts stay
    keep = held + want_count.astype(int)
    alloc.trim((u32(held, device).view(torch.int32) + count.view(torch.int32)).view(torch.uint32))
    assert alloc.positions.cpu().numpy().tolist() == keep.tolist()
    assert alloc.row_blocks.cpu().numpy().tolist() == (-(-keep // BS)).tolist()
    for s in range(3):
        m.next_pos[s] -= 4 - int(want_count[s])
        for j in range(KVH):
            del m.tokens[s][j][keep[s]:]
    slots, ctx = alloc.step()
    assert ctx.cpu().numpy().tolist() == (keep + 1).tolist()
    q = m.append([1, 1, 1], slots)
    out = vpa.paged_attention(q, None, None, m.kc, m.vc, alloc.block_tables, ctx, None,
                              int(keep.max()) + 1, SCALE, 1.0, None)
    m.check_attention(out, q, [1, 1, 1])


def test_trim(device):
    """Rows go back to fewer tokens, none, or stay; the freed blocks serve others."""
    alloc = vpa.DeviceBlockAllocator(20, 16, 4, 8, device)
    assert alloc.allocate(u32([33, 16, 5, 128], device)).all()
    assert int(alloc.free_ring_state[1]) == 19 - (3 + 1 + 1 + 8)
    first = alloc.block_tables.cpu().numpy().copy()
    alloc.trim(u32([32, 0, 5, 17], device))
    assert alloc.positions.cpu().numpy().tolist() == [32, 0, 5, 17]
    assert alloc.row_blocks.cpu().numpy().tolist() == [2, 0, 1, 2]
    assert int(alloc.free_ring_state[1]) == 19 - 5
    slots, ctx = alloc.step()
    assert ctx.cpu().numpy().tolist() == [33, 1, 6, 18]
    got = slots.cpu().numpy()
    assert got[2] == first[2, 0] * 16 + 5 and got[3] == first[3, 1] * 16 + 1
    assert alloc.row_blocks.cpu().numpy().tolist() == [3, 1, 1, 2]
    with pytest.raises(vpa.VpaError, match="num_tokens"):
        alloc.trim(torch.zeros(4, dtype=torch.int32, device=device))
    with pytest.raises(vpa.VpaError, match="num_tokens"):
        alloc.trim(u32([1, 2, 3], device))


def test_loop_on_a_side_stream(device):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        test_loop(device)
    torch.cuda.current_stream().wait_stream(side)


class Step:
    """A decode step of a bounded cache: append, attention, weights, the cut to 40 tokens,
    verification of two drafts; every buffer fixed, so that it can be captured."""

    def __init__(self, device):
        gen = torch.Generator().manual_seed(8)
        rand = lambda *s: torch.randn(s, generator=gen).to(device)  # noqa: E731
        self.alloc = vpa.DeviceBlockAllocator(20, BS, 3, 4, device)
        assert self.alloc.allocate(u32([50, 23, 39], device)).all()
        self.alloc.positions.copy_(u32([50, 23, 39], device))
        self.kc, self.vc = rand(20, KVH, D // 4, BS, 4), rand(20, KVH, D, BS)
        self.scores = rand(3, KVH, 64).abs()
        self.q, self.k, self.v = rand(3, H, D), rand(3, KVH, D), rand(3, KVH, D)
        self.pos = torch.tensor([[50, 23, 39]], device=device)
        self.inv_freq, self.axes = vpa.rotary_frequencies(D, 1e4, device)
        self.target, self.draft = 2 * rand(3, 3, 900), 2 * rand(3, 2, 900)
        self.ids = u32(self.draft.argmax(-1).cpu().numpy(), device)
        self.u = torch.rand((3, 3), generator=gen).to(device)
        self.out = self.verified = None

    def __call__(self):
        a = self.alloc
        slots, ctx = a.step()
        q = vpa.rotary_reshape_and_cache(self.q, self.k, self.v, self.pos, self.inv_freq, self.axes,
                                         None, None, self.kc, self.vc, slots)
        self.out = vpa.paged_attention(q, None, None, self.kc, self.vc, a.block_tables, ctx, None, 64,
                                       SCALE, 1.0, None)
        vpa.paged_attention_weights(q, self.kc, None, a.block_tables, ctx, SCALE, self.scores,
                                    max_context_len=64)
        lens, self.kept = vpa.evict_kv_cache(self.kc, self.vc, self.scores, a.block_tables, ctx, 40,
                                             keep_first=2, keep_last=4, max_context_len=64)
        a.trim(lens)
        self.verified = vpa.verify_draft_tokens(self.target, self.ids, self.u[:, :2], self.u[:, 2],
                                                draft_logits=self.draft)
        self.pos.add_(1)

    def state(self):
        a = self.alloc
        return [self.out, self.kc, self.vc, self.scores, self.kept, self.pos, *self.verified,
                a.positions, a.row_blocks, a.block_tables, a.free_ring, a.free_ring_state]

    def inputs(self, i):
        for x, scale in ((self.q, 1.0), (self.k, 1.1), (self.target, 0.9)):
            x.copy_(torch.roll(x, i + 1, -1) * scale)
        self.u.copy_(torch.roll(self.u, 1, 0))


def test_step_captured_and_replayed(device):
    """Two captured steps of two states, replayed in turn, against the same steps run
    eagerly between the replays."""
    eager, graphs, steps = Step(device), [], [Step(device), Step(device)]
    Step(device)()  # (first use outside a capture)
    torch.cuda.synchronize()
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s()
        graphs.append(g)
    for i in range(5):
        eager()
        for g, s in zip(graphs, steps):
            g.replay()
        torch.cuda.synchronize()
        for s in steps:
            for x, y in zip(s.state(), eager.state()):
                x, y = (t.view(torch.int32) if t.dtype == torch.uint32 else t for t in (x, y))
                assert torch.equal(x, y), i
        for s in (eager, *steps):
            s.inputs(i)
    assert eager.alloc.positions.cpu().numpy().tolist() == [40, 28, 40]
    assert eager.alloc.row_blocks.cpu().numpy().tolist() == [3, 2, 3]


def refusals(device):
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
    w = lambda *s: z(*s, dtype=torch.int32).view(torch.uint32)  # noqa: E731
    q, k, pos, f = z(5, 4, 64), z(5, 2, 64), z(1, 5, dtype=torch.int64), z(32, dtype=torch.float64)
    kc, vc, slots = z(9, 2, 16, 16, 4), z(9, 2, 64, 16), z(5, dtype=torch.int64)
    bt, cl, sc = w(3, 4), w(3), z(3, 2, 64)
    t, ids, au, su = z(3, 3, 50), w(3, 2), z(3, 2), z(3)
    rq, rc = vpa.rotary_qk, vpa.rotary_reshape_and_cache
    pw, ev, vd = vpa.paged_attention_weights, vpa.evict_kv_cache, vpa.verify_draft_tokens
    cache = (None, None, kc, vc)
    return [
        ("must be \\[T, heads, D\\]", lambda: rq(q[0], k, pos, f)),
        ("k must be", lambda: rq(q, k[:4], pos, f)),
        ("k must be", lambda: rq(q, k.half(), pos, f)),
        ("positions", lambda: rq(q, k, pos[:, :4], f)),
        ("positions", lambda: rq(q, k, pos.int(), f)),
        ("inv_freq", lambda: rq(q, k, pos, f.float())),
        ("axes", lambda: rq(q, k, pos, f, z(31, dtype=torch.uint8))),
        ("q_norm", lambda: rq(q, k, pos, f, q_norm=z(64).half())),
        ("k_norm", lambda: rq(q, k, pos, f, k_norm=z(32))),
        ("out_q", lambda: rq(q, k, pos, f, out_q=z(5, 4, 32))),
        ("rotary_dim", lambda: rq(q, k, pos, z(33, dtype=torch.float64))),
        ("num_axes", lambda: rq(q, k, z(5, 5, dtype=torch.int64), f)),
        ("q, k and v", lambda: rc(q, k, z(5, 2, 32), pos, f, None, *cache, slots)),
        ("one dtype", lambda: rc(q, k, k.half(), pos, f, None, *cache, slots)),
        ("slot_mapping", lambda: rc(q, k, k, pos, f, None, *cache, slots[:4])),
        ("differs", lambda: rc(q.half(), k.half(), k.half(), pos, f, None, *cache, slots)),
        ("out must", lambda: rc(q, k, k, pos, f, None, *cache, slots, out=k)),
        ("a row per sequence", lambda: pw(q, kc, None, bt, cl, 1.0, sc, max_context_len=64)),
        ("q must be", lambda: pw(q[:3, :, :32], kc, None, bt, cl, 1.0, sc, max_context_len=64)),
        ("cu_seqlens_q", lambda: pw(q, kc, None, bt, cl, 1.0, sc, cu_seqlens_q=w(3), max_query_len=2,
                                    max_context_len=64)),
        ("scores", lambda: pw(q[:3], kc, None, bt, cl, 1.0, sc[:, :, :60], max_context_len=64)),
        ("scores", lambda: pw(q[:3], kc, None, bt, cl, 1.0, sc.half(), max_context_len=64)),
        ("contiguous along", lambda: pw(q[:3], kc, None, bt, cl, 1.0, z(3, 2, 128)[..., ::2],
                                        max_context_len=64)),
        ("overlap", lambda: pw(q[:3], kc, None, bt, cl, 1.0, z(1, 2, 64).expand(3, 2, 64),
                               max_context_len=64)),
        ("too small", lambda: pw(q[:3], kc, None, bt, cl, 1.0, z(3, 2, 65), max_context_len=65)),
        ("bytes needed", lambda: pw(q[:3], kc, None, bt, cl, 1.0, sc, max_context_len=64,
                                    workspace=z(1))),
        ("block_tables", lambda: ev(kc, vc, sc, bt.view(torch.int32), cl, 8, max_context_len=64)),
        ("context_lens", lambda: ev(kc, vc, sc, bt, cl[:2], 8, max_context_len=64)),
        ("budget", lambda: ev(kc, vc, sc, bt, cl, 0, max_context_len=64)),
        ("budget", lambda: ev(kc, vc, sc, bt, cl, 8, keep_first=5, keep_last=4, max_context_len=64)),
        ("new_context_lens", lambda: ev(kc, vc, sc, bt, cl, 8, max_context_len=64,
                                        new_context_lens=cl)),
        ("kept", lambda: ev(kc, vc, sc, bt, cl, 8, max_context_len=64, kept=w(3, 2, 7))),
        ("shape mismatch", lambda: ev(kc, vc[:8], sc, bt, cl, 8, max_context_len=64)),
        ("target_logits", lambda: vd(t[0], ids, au, su)),
        ("draft_ids", lambda: vd(t, ids[:, :1], au, su)),
        ("accept_u", lambda: vd(t, ids, au.double(), su)),
        ("sample_u", lambda: vd(t, ids, au, su[:2])),
        ("draft_logits", lambda: vd(t, ids, au, su, draft_logits=t)),
        ("temperature", lambda: vd(t, ids, au, su, temperature=z(2))),
        ("num_drafts", lambda: vd(t, ids, au, su, num_drafts=z(3, dtype=torch.int32))),
        ("out must", lambda: vd(t, ids, au, su, out=(w(3, 2), w(3)))),
        ("exceeds 64", lambda: vd(z(1, 66, 8), w(1, 65), z(1, 65), z(1))),
        ("dtype", lambda: vd(t.double(), ids, au, su)),
        ("GPU only", lambda: vd(t, ids.cpu(), au, su)),
    ]


@pytest.mark.parametrize("i", range(44))
def test_wrong_tensors_are_refused(device, i):
    cases = refusals(device)
    assert len(cases) == 44
    needle, call = cases[i]
    with pytest.raises(vpa.VpaError, match=needle):
        call()
