"""The block-scaled cache, forked rows, compaction and adjusted logits as a serving loop runs
them: through DeviceDecodeStep against a host model, captured into replayed graphs, on a side
stream."""

import numpy as np
import pytest
import torch

import vpa
from tests import _serving_oracle as ref
from tests._util import i64, u32

pytestmark = pytest.mark.gpu

H, KVH, D, BS, NB, ROWS, V, LAYERS = 4, 2, 64, 16, 64, 6, 500, 2
EOS = 499


class Loop:
    """Two layers over block-scaled caches; q, k, v and logits are functions of the row's
    tokens and position, so the host can follow."""

    def __init__(self, device):
        self.device = device
        self.step = vpa.DeviceDecodeStep(ROWS, NB, BS, 96, H, D, [EOS], 40, device)
        self.caches = []
        for _ in range(LAYERS):
            kc = torch.full((NB, KVH, D // 16, BS, 16), 0x7F, dtype=torch.uint8, device=device)
            vc = torch.full((NB, KVH, D, BS), 0xFF, dtype=torch.uint8, device=device)
            self.caches.append((kc, vc) + vpa.block_scales(NB, KVH, device))
        rng = np.random.default_rng(0)
        self.table = torch.from_numpy(rng.standard_normal((V, LAYERS, (H + 2 * KVH) * D)).astype(
            np.float32)).to(device)
        self.head = torch.from_numpy(rng.standard_normal((V, V)).astype(np.float32)).to(device)
        self.out = torch.empty((ROWS, H, D), device=device)
        self.rep = torch.full((ROWS,), 1.5, device=device)
        self.pres = torch.full((ROWS,), 0.7, device=device)
        bits = rng.random((1, V)) < 0.5
        bits[0, EOS] = False
        words = np.packbits(np.pad(bits, ((0, 0), (0, 12))), axis=1, bitorder="little").view(np.uint32)
        self.mask, self.allowed = bits[0], u32(words, device)
        self.rules = dict(repetition=self.rep, presence=self.pres, allowed=self.allowed,
                          allowed_rows=u32(np.zeros(ROWS), device))
        # the host's side: each row's cached tokens and generated ids
        self.tokens, self.generated, self.pending = [[] for _ in range(ROWS)], [[] for _ in range(ROWS)], [0] * ROWS

    @property
    def buffers(self):
        return [t for layer in self.caches for t in layer]

    def rows(self, ids, layer):
        x = self.table[ids.long(), layer]
        return (x[:, :H * D].view(-1, H, D), x[:, H * D:(H + KVH) * D].view(-1, KVH, D),
                x[:, (H + KVH) * D:].view(-1, KVH, D))

    def admit(self, prompts):
        lens = [len(p) for p in prompts] + [0] * (ROWS - len(prompts))
        ok = self.step.admit(u32(lens, self.device))
        assert ok.cpu().all()
        tables = self.step.allocator.block_tables.cpu().numpy()
        for r, p in enumerate(prompts):
            t = np.arange(len(p))
            slots = i64(tables[r, t // BS].astype(np.int64) * BS + t % BS, self.device)
            for layer, (kc, vc, ks, vs) in enumerate(self.caches):
                _, k, v = self.rows(torch.tensor(p, device=self.device), layer)
                vpa.reshape_and_cache_block_scaled(k, v, ks, vs, kc, vc, slots)
            self.tokens[r] = list(p)
        self.step.tokens.finished.copy_(torch.tensor([int(n == 0) for n in lens], dtype=torch.uint8))

    def decode(self):
        """One step on the device."""
        kc, vc = self.caches[0][:2]
        self.step.begin(kc, vc, torch.float32)
        ids = self.step.tokens.input_ids.view(torch.int32)
        x = 0
        for layer, (kc, vc, ks, vs) in enumerate(self.caches):
            q, k, v = self.rows(ids, layer)
            self.step.layer(q, k, v, kc, vc, self.out, ks, vs)
            x = x + self.out.sum((1, 2))
        logits = self.head[ids.long()] + 0.01 * x[:, None]
        self.step.end(logits, **self.rules)
        return logits

    def follow(self, live):
        """The same step on the host for rows `live`; checks the last layer's attention
        and the chosen ids."""
        torch.cuda.synchronize()
        lens = self.step.allocator.context_lens.cpu().numpy()
        out = self.out.double().cpu().numpy()
        chosen = self.step.tokens.next_ids.cpu().numpy()
        head = self.head.cpu().numpy()
        tables = self.step.allocator.block_tables.cpu().numpy()
        for r in live:
            self.generated[r].append(self.pending[r])
            self.tokens[r].append(self.pending[r])
            n = len(self.tokens[r])
            assert lens[r] == n
            kc, vc, ks, vs = (t.cpu().numpy() for t in self.caches[-1])
            q, k, v = (t.cpu().numpy().astype(np.float64) for t in self.rows(
                torch.tensor(self.tokens[r], device=self.device), LAYERS - 1))
            # what the cache holds is each token's row within E4M3's half step, or below
            # its normal range the half steps 2^-10 s of the scales so far, each at most
            # half of the next: under 2^-9 s together
            t = np.arange(n)
            blk = tables[r, t // BS].astype(np.int64)
            for got, want, s in ((kc[blk, :, :, t % BS].reshape(n, KVH, D), k, ks[blk]),
                                 (vc[blk, :, :, t % BS], v, vs[blk])):
                err = np.abs(ref.e4m3_value(got) * s[..., None] - want)
                assert np.all(err <= 2.0 ** -4 * np.abs(want) + 2.0 ** -9 * s[..., None])
            want, *rest = ref.attention(q[n - 1:n].astype(np.float32), ks, vs, kc, vc, tables[r:r + 1],
                                        [n], D ** -0.5, eps=1e-6)
            bound = ref.attention_bound(want, *rest, D, n, 2.0 ** -24)
            assert np.all(np.abs(out[r] - want[0]) <= bound[0])
            row, _ = ref.adjust(head[self.pending[r]], self.generated[r], rep=1.5, pres=0.7,
                                mask=self.mask)
            # (all logits of a row are moved by the same sum of outputs, which may turn a
            # penalty's direction next to zero: the choice is among the best)
            assert row[chosen[r]] >= np.nanmax(row) - 0.2
            self.pending[r] = int(chosen[r])


def test_a_loop_with_forks_and_compaction(device):
    rng = np.random.default_rng(1)
    loop = Loop(device)
    loop.admit([list(rng.integers(0, V - 1, size=n)) for n in (37, 16)])
    live = [0, 1]
    for _ in range(3):
        loop.decode()
        loop.follow(live)
    # row 0 goes on as three, row 1 as two
    ok = loop.step.fork(u32([0, 0, 1, 0], device), u32([2, 3, 4, 2], device), loop.buffers)
    assert ok.cpu().tolist() == [1, 1, 1, 0]
    for a, b in ((0, 2), (0, 3), (1, 4)):
        loop.tokens[b], loop.generated[b] = list(loop.tokens[a]), list(loop.generated[a])
        loop.pending[b] = loop.pending[a]
    # the forks go on with other tokens than their sources
    for r, t in ((2, 11), (3, 12), (4, 13)):
        loop.pending[r] = t
        loop.step.tokens.next_ids.view(torch.int32)[r] = t
    live = [0, 1, 2, 3, 4]
    for _ in range(BS + 2):  # past a block's end
        loop.decode()
        loop.follow(live)
    assert int(loop.step.allocator.shared.view(torch.int32).sum()) > 0
    # row 0 ends: its shared blocks stay with rows 2 and 3
    loop.step.tokens.finished[0] = 1
    keep = np.full(ROWS, 99, np.uint32)
    keep[0] = 0
    loop.step.allocator.release(u32(keep, device))
    live = [1, 2, 3, 4]
    src, dst, count = loop.step.allocator.compact(loop.buffers)
    assert int(count.cpu()[0]) > 0
    held = loop.step.allocator.block_tables.cpu().numpy()
    n = loop.step.allocator.row_blocks.cpu().numpy()
    used = {int(b) for r in range(ROWS) for b in held[r, :n[r]]}
    assert used == set(range(1, len(used) + 1))
    for _ in range(4):
        loop.decode()
        loop.follow(live)
    # rejected tokens taken back in a row of its own blocks, and below a shared one
    back = [len(t) for t in loop.tokens]
    back[2], back[3] = len(loop.tokens[2]) - 3, 20
    back[0] = 0
    slots = loop.step.allocator.slot_mapping
    loop.step.allocator.trim(u32(back, device), buffers=loop.buffers)
    assert loop.step.allocator.ok.cpu().all() and slots is loop.step.allocator.slot_mapping
    for r in (2, 3):
        loop.tokens[r] = loop.tokens[r][:back[r]]
    for _ in range(3):
        loop.decode()
        loop.follow(live)


def test_graph_of_a_step_replayed(device):
    """A captured step (append, attention, rules, choice) replayed with eager work
    between, against the same steps run eagerly."""
    rng = np.random.default_rng(2)
    prompts = [list(rng.integers(0, V - 1, size=n)) for n in (20, 5, 33)]
    results = []
    for captured in (False, True):
        loop = Loop(device)
        loop.step.allocator.enable_sharing()
        loop.admit(prompts)
        got = []
        loop.decode()  # (workspaces and libraries are ready)
        got.append(loop.step.tokens.next_ids.clone())
        graph = None
        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                loop.decode()
        for i in range(6):
            if captured:
                graph.replay()
            else:
                loop.decode()
            torch.cuda.synchronize()
            got.append(loop.step.tokens.next_ids.clone())
            if i == 2:  # eager work between: a fork
                ok = loop.step.fork(u32([0, 2], device), u32([3, 4], device), loop.buffers)
                assert ok.cpu().all()
        got += [loop.out.clone()] + [t.clone() for t in loop.buffers]
        results.append(got)
    for i, (a, b) in enumerate(zip(*results)):
        if a.is_floating_point():
            assert torch.equal(a.view(torch.int32), b.view(torch.int32)), i
        else:
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i


def test_pages_in_a_replayed_graph(device):
    """Fork, release and compaction captured together: every replay equals the eager run."""
    def fresh():
        a = vpa.DeviceBlockAllocator(50, 8, 6, 6, device)
        a.enable_sharing()
        target = u32([20, 33, 7, 0, 0, 0], device)
        a.allocate(target)
        a.positions.copy_(target)
        pool = torch.arange(50 * 64, device=device, dtype=torch.float32).view(50, 64)
        return a, [pool]

    keep = u32([99, 0, 99, 0, 99, 0], device)
    again = u32([0, 33, 0, 0, 0, 0], device)
    src, dst = u32([0, 2, 1], device), u32([3, 4, 5], device)

    def turn(a, buffers):
        a.fork(src, dst, buffers)
        a.release(keep)
        a.compact(buffers)
        a.allocate(again)

    states = []
    for captured in (False, True):
        a, buffers = fresh()
        steps = []
        if captured:
            warm, wb = fresh()
            turn(warm, wb)
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                turn(a, buffers)
        for _ in range(4):
            if captured:
                graph.replay()
            else:
                turn(a, buffers)
            torch.cuda.synchronize()
            steps += [t.clone() for t in (a.block_tables, a.row_blocks, a.positions, a.shared,
                                          a.free_ring, a.free_ring_state)] + [buffers[0].clone()]
        states.append(steps)
    for i, (x, y) in enumerate(zip(*states)):
        assert torch.equal(x.view(torch.int32), y.view(torch.int32)), i


def test_forking_under_capture_needs_sharing_enabled(device):
    a = vpa.DeviceBlockAllocator(10, 8, 2, 3, device)
    pool = [torch.zeros((10, 4), device=device)]
    src, dst = u32([0], device), u32([1], device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device=device)  # (a graph of nothing is refused by some versions)
        with pytest.raises(vpa.VpaError, match="before the graph"):
            a.fork(src, dst, pool)


def test_side_stream(device):
    """Every call on a stream of its own equals the call on the current one."""
    rng = np.random.default_rng(4)
    nb, lens = 40, [200, 90]
    kc = torch.randint(0, 100, (nb, KVH, D // 16, BS, 16), dtype=torch.uint8, device=device)
    vc = torch.randint(0, 100, (nb, KVH, D, BS), dtype=torch.uint8, device=device)
    ks, vs = torch.full((nb, KVH), 0.01, device=device), torch.full((nb, KVH), 0.02, device=device)
    tables = u32(rng.permutation(np.arange(1, 27)).reshape(2, 13), device)
    k = torch.randn((2, KVH, D), device=device)
    q = torch.randn((2, H, D), device=device)
    logits = torch.randn((2, V), device=device)
    gen, rep = u32(rng.integers(0, V, size=(2, 30)), device), torch.full((2,), 1.3, device=device)
    slots = i64([30 * BS + 1, 31 * BS], device)

    def calls():
        c = [t.clone() for t in (kc, vc, ks, vs, logits)]
        vpa.reshape_and_cache_block_scaled(k, k, c[2], c[3], c[0], c[1], slots)
        out = vpa.paged_attention_block_scaled(q, c[2], c[3], c[0], c[1], tables, u32(lens, device),
                                               0.1, max_context_len=200)
        vpa.adjust_logits(c[4], gen, repetition=rep)
        vpa.copy_blocks(c[:4], tables[0, :3], u32([35, 36, 37], device))
        return c + [out]

    want = calls()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = calls()
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_a_step_over_a_cache_of_one_scale(device):
    """One-element scales are an fp8 cache's, whatever their shape."""
    rng = np.random.default_rng(6)
    step = vpa.DeviceDecodeStep(2, 8, BS, 64, H, D, [EOS], 8, device)
    assert step.admit(u32([5, 20], device)).cpu().all()
    q, k, v = (torch.from_numpy(rng.standard_normal((2, n, D)).astype(np.float32)).to(device)
               for n in (H, KVH, KVH))
    outs = []
    for shape in ((1,), (1, 1)):
        kc = torch.zeros((8, KVH, D // 16, BS, 16), dtype=torch.uint8, device=device)
        vc = torch.zeros((8, KVH, D, BS), dtype=torch.uint8, device=device)
        if not outs:
            step.begin(kc, vc, torch.float32)
        one = torch.full(shape, 0.25, device=device)
        outs.append(torch.empty((2, H, D), device=device))
        step.layer(q, k, v, kc, vc, outs[-1], one, one)
    torch.cuda.synchronize()
    assert outs[0].any() and torch.equal(outs[0], outs[1])


def test_a_block_scaled_step_needs_no_work_list(device):
    rng = np.random.default_rng(7)
    prompts = [list(rng.integers(0, V - 1, size=n)) for n in (20, 5)]
    chosen = []
    for skip in (False, True):
        loop = Loop(device)
        if skip:
            begin = loop.step.begin
            loop.step.begin = lambda *a: begin(*a, block_scaled=True)
        loop.admit(prompts)
        for _ in range(4):
            loop.decode()
        torch.cuda.synchronize()
        chosen.append(loop.step.tokens.next_ids.cpu().numpy()[:2].tolist())
    assert chosen[0] == chosen[1]
