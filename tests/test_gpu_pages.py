"""GPU tests of forked, released, unshared and compacted blocks and of their copies:
whole numbers and bytes, equal to a host model that takes one row and block at a time."""

import numpy as np
import pytest
import torch

import vpa
from tests import _serving_oracle as ref
from tests._util import u32

pytestmark = pytest.mark.gpu


class Both:
    """The device allocator and the model, with two small pools whose bytes follow."""

    def __init__(self, device, nb, bs, rows, cols, seed=0):
        self.device, self.rng = device, np.random.default_rng(seed)
        self.dev = vpa.DeviceBlockAllocator(nb, bs, rows, cols, device)
        self.ref = ref.Pages(nb, bs, rows, cols)
        self.buffers = [torch.from_numpy(self.rng.integers(0, 255, (nb, 3, 16), dtype=np.uint8)).to(device),
                        torch.from_numpy(self.rng.standard_normal((nb, 5)).astype(np.float32)).to(device)]
        self.want = [b.cpu().numpy().copy() for b in self.buffers]
        self.dev.enable_sharing()

    def shuffle(self):
        """The ring's ids in another order."""
        ids = self.rng.permutation(np.arange(1, self.ref.nb)).astype(np.uint32)
        self.ref.ring[:len(ids)] = ids
        self.dev.free_ring.copy_(u32(self.ref.ring, self.device))

    def copied(self, pairs):
        for b in self.want:
            old = b.copy()
            for src, dst in pairs:
                b[dst] = old[src]

    def allocate(self, target):
        self.dev.allocate(u32(target, self.device))
        self.dev.positions.copy_(u32(target, self.device))
        self.ref.allocate(target)
        self.ref.positions[:] = target

    def fork(self, src, dst):
        ok = self.dev.fork(u32(src, self.device), u32(dst, self.device), self.buffers)
        want, pairs = self.ref.fork(src, dst)
        self.copied(pairs)
        assert ok.cpu().tolist() == [int(x) for x in want]
        return want

    def release(self, keep):
        self.dev.release(u32(keep, self.device))
        self.ref.release(keep)

    def trim(self, tokens):
        self.dev.trim(u32(tokens, self.device), buffers=self.buffers)
        self.ref.positions[:] = tokens
        self.ref.release(-(-np.asarray(tokens) // self.ref.bs))
        ok, pairs = self.ref.unshare()
        self.copied(pairs)
        assert self.dev.ok.cpu().tolist() == [int(x) for x in ok]

    def compact(self):
        src, dst, count = self.dev.compact(self.buffers)
        pairs = self.ref.compact()
        self.copied(pairs)
        n = int(count.cpu()[0])
        assert list(zip(src[:n].cpu().tolist(), dst[:n].cpu().tolist())) == pairs

    def check(self):
        torch.cuda.synchronize()
        d, r = self.dev, self.ref
        held = d.row_blocks.cpu().numpy()
        assert np.array_equal(held, r.held)
        tables = d.block_tables.cpu().numpy()
        for row in range(len(held)):
            assert np.array_equal(tables[row, :held[row]], r.tables[row, :held[row]]), row
        assert np.array_equal(d.positions.cpu().numpy(), r.positions)
        assert np.array_equal(d.shared.cpu().numpy(), r.shared)
        state = d.free_ring_state.cpu().numpy()
        assert list(state) == [r.head, r.count]
        at = (r.head + np.arange(r.count)) % r.nb
        assert np.array_equal(d.free_ring.cpu().numpy()[at], r.ring[at])
        for got, want in zip(self.buffers, self.want):
            assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("bs", [1, 8, 16])
def test_fork_shares_whole_blocks_and_copies_the_last(device, bs):
    b = Both(device, 60, bs, 12, 9)
    b.shuffle()
    b.allocate([3 * bs, 5 * bs + bs // 2 + 1, 1, 0] + [0] * 8)
    b.check()
    # an empty row's copy is empty; one source twice; a whole-block row; refused ones
    assert b.fork([1, 1, 0, 3, 2, 2, 99, 1, 4294967295], [4, 5, 6, 7, 8, 0, 9, 4, 10]) == \
        [True, True, True, True, True, False, False, False, False]
    b.check()
    b.fork([4, 5], [9, 10])  # copies of copies
    b.check()
    b.release([99] * 4 + [0] * 8)
    b.check()
    assert not b.ref.shared.any()
    b.release([0] * 12)
    b.check()
    assert b.ref.count == 59


def test_sources_are_read_as_they_stand(device):
    """A fork's target that is another fork's source still counts as empty there."""
    b = Both(device, 30, 4, 5, 6)
    b.allocate([10, 0, 0, 0, 0])
    assert b.fork([0, 1, 0, 2], [1, 2, 3, 2]) == [True, True, True, False]
    b.check()


def test_fork_without_blocks_left(device):
    b = Both(device, 8, 4, 8, 4)
    b.allocate([6, 8, 5] + [0] * 5)  # 2 + 2 + 2 blocks of 7
    got = b.fork([0, 2, 1, 0], [3, 4, 5, 6])  # one block left; row 1 needs none
    assert got == [True, False, True, False]
    b.check()
    b.release([0, 99, 99, 99, 99, 99, 99, 99])
    b.check()


def test_many_forks(device):
    b = Both(device, 2000, 8, 1025, 20)
    b.shuffle()
    b.allocate([150] + [0] * 1024)
    b.fork([0] * 1024, list(range(1, 1025)))
    b.check()
    keep = [0 if r % 3 else 99 for r in range(1025)]
    b.release(keep)
    b.check()
    b.release([0] * 1025)
    b.check()


@pytest.mark.parametrize("rows,tokens", [(200, 164), (200, 165), (512, 80), (1024, 40), (1000, 99)])
def test_release_entries_beyond_a_lane_s_few(device, rows, tokens):
    """About 4096 entries of one list of rows, more, and blocks of their own in between."""
    b = Both(device, 7000, 8, rows, 22, seed=rows)
    b.shuffle()
    b.allocate([tokens, tokens // 2] + [0] * (rows - 2))
    b.fork(list(b.rng.integers(0, 2, size=rows - 2)), list(range(2, rows)))
    b.check()
    b.release(list(b.rng.integers(0, 3, size=rows)))
    b.check()
    b.release([0] * rows)
    b.check()
    assert b.ref.count == 6999


def test_release_more_rows_than_a_pass_takes(device):
    b = Both(device, 6000, 4, 2100, 5, seed=2)
    b.allocate(list(b.rng.integers(0, 9, size=2000)) + [0] * 100)
    src = b.rng.integers(0, 2000, size=100)
    b.fork(list(src), list(range(2000, 2100)))
    b.check()
    b.release(list(b.rng.integers(0, 3, size=2100)))
    b.check()


def test_release_keeps_of_any_size(device):
    b = Both(device, 40, 4, 3, 8)
    b.allocate([20, 9, 0])
    b.release([0xFFFFFFFF, 1, 0xFFFFFFFF])
    b.check()
    b.release([0, 0xFFFFFFF0, 0])
    b.check()


def test_trim_below_a_shared_block(device):
    b = Both(device, 40, 8, 6, 6)
    b.shuffle()
    b.allocate([24, 0, 0, 0, 0, 0])
    b.fork([0, 0, 0], [1, 2, 3])
    b.check()
    b.trim([24, 20, 17, 16, 0, 0])  # rows 1 and 2 end inside a block that others hold
    b.check()
    b.trim([20, 20, 12, 3, 0, 0])
    b.check()
    # nobody shares any more where only one row is left
    b.release([0, 0, 0, 99, 0, 0])
    b.trim([0, 0, 0, 2, 0, 0])
    b.check()


def test_trim_without_blocks_left(device):
    b = Both(device, 7, 8, 3, 3)
    b.allocate([24, 0, 0])
    b.fork([0, 0], [1, 2])
    b.ref.count = 0
    b.dev.free_ring_state.copy_(u32([b.ref.head, 0], device))
    b.trim([24, 20, 20])
    b.check()


def test_trim_needs_buffers_where_blocks_are_shared(device):
    b = Both(device, 10, 8, 2, 3)
    with pytest.raises(vpa.VpaError, match="buffers"):
        b.dev.trim(u32([0, 0], device))


@pytest.mark.parametrize("nb", [2, 3, 33, 65, 1000, 40000, 65536, 65537, 200000])
def test_compact(device, nb):
    rows = 6
    b = Both(device, nb, 4, rows, min(max(2, nb // 4), 30000), seed=nb)
    b.compact()  # nothing in use
    b.check()
    b.shuffle()
    b.allocate([4 * int(n) for n in b.rng.integers(0, min(max(2, nb // 7), 29000), size=rows)])
    b.fork([0, 1], [4, 5])  # (refused where the rows hold blocks)
    b.check()
    b.compact()
    b.check()
    b.release([0, 99999, 0, 99999, 1, 99999])
    b.compact()
    b.check()
    b.compact()  # no moves
    b.check()
    if nb > 30:
        b.allocate([4 * (int(n) + 1) for n in b.ref.held])
        b.check()


def test_compact_a_full_pool_and_blocks_outside_the_tables(device):
    b = Both(device, 17, 4, 2, 16)
    b.allocate([64, 0])
    assert b.ref.count == 0
    b.compact()
    b.check()
    b.release([0, 0])
    b.shuffle()
    for _ in range(3):  # a caller's own blocks, in no table
        b.ref.take()
    b.dev.free_ring_state.copy_(u32([b.ref.head, b.ref.count], device))
    b.allocate([20, 8])
    b.compact()
    b.check()


def test_random_sequences(device):
    for seed in range(4):
        rng = np.random.default_rng(100 + seed)
        b = Both(device, int(rng.integers(40, 200)), int(rng.choice([1, 4, 16])), 12, 10, seed)
        b.shuffle()
        for _ in range(25):
            op = rng.integers(5)
            if op == 0:
                b.allocate(np.maximum(b.ref.positions, rng.integers(0, 10 * b.ref.bs, size=12) *
                                      (rng.random(12) < 0.4)).astype(np.int64))
                # (positions of rows that found no blocks stay within what they hold)
                fit = np.minimum(b.ref.positions, b.ref.held * b.ref.bs)
                b.ref.positions[:] = fit
                b.dev.positions.copy_(u32(fit, device))
            elif op == 1:
                n = int(rng.integers(1, 6))
                b.fork(list(rng.integers(0, 13, size=n)), list(rng.integers(0, 13, size=n)))
            elif op == 2:
                keep = np.where(rng.random(12) < 0.4, rng.integers(0, 10, size=12), 99)
                b.release(list(keep))
                fit = np.minimum(b.ref.positions, b.ref.held * b.ref.bs)
                b.ref.positions[:] = fit
                b.dev.positions.copy_(u32(fit, device))
            elif op == 3:
                b.trim(np.where(rng.random(12) < 0.5, b.ref.positions,
                                (b.ref.positions * rng.random(12)).astype(np.int64)))
            else:
                b.compact()
            b.check()


# ---- copies -------------------------------------------------------------------


def test_copy_blocks_of_any_size(device):
    """Sizes and strides that go by 16 bytes, by 4 and by 1; views with gaps; more buffers
    than one launch takes; pairs past the pool, of one block, behind the count."""
    rng = np.random.default_rng(0)
    nb = 50
    wide = torch.from_numpy(rng.integers(0, 255, (nb, 4096 + 48), dtype=np.uint8)).to(device)
    buffers = [wide[:, 16:16 + 4096], wide[:, 4128:4132],
               torch.from_numpy(rng.integers(0, 255, (nb, 7), dtype=np.uint8)).to(device),
               torch.from_numpy(rng.standard_normal((nb, 8, 3)).astype(np.float32)).to(device),
               torch.from_numpy(rng.integers(0, 9, (nb, 33000), dtype=np.uint8)).to(device),
               torch.zeros((nb, 0), device=device)]
    buffers += [torch.from_numpy(rng.integers(0, 99, (nb, 16), dtype=np.uint8)).to(device)
                for _ in range(200)]
    want = [b.cpu().numpy().copy() for b in buffers]
    src, dst = [3, 3, 49, 7, 60, 8, 9, 11], [4, 5, 0, 7, 6, 4294967295, 10, 12]
    count = u32([7], device)
    vpa.copy_blocks(buffers, u32(src, device), u32(dst, device), count)
    torch.cuda.synchronize()
    for a, b in list(zip(src, dst))[:7]:
        if a < nb and b < nb:
            for w in want:
                w[b] = w[a]
    for k, (g, w) in enumerate(zip(buffers, want)):
        assert np.array_equal(g.cpu().numpy(), w), k
    rest = wide.cpu().numpy()
    assert np.array_equal(rest[:, 16:4112], want[0])


def test_copy_without_pairs_or_buffers(device):
    b = torch.arange(12, device=device, dtype=torch.float32).view(3, 4)
    none = u32(np.zeros(0, np.uint32), device)
    vpa.copy_blocks([b], none, none)
    vpa.copy_blocks([], u32([1], device), u32([2], device))
    vpa.copy_blocks([b], u32([1], device), u32([2], device), u32([0], device))
    assert torch.equal(b, torch.arange(12, device=device, dtype=torch.float32).view(3, 4))


@pytest.mark.parametrize("n", [1, 191, 192, 193, 400])
def test_any_number_of_buffers(device, n):
    """More than a launch takes, of sizes in vectors, words and bytes."""
    rng = np.random.default_rng(n)
    host = [rng.integers(0, 255, (6, (16, 4, 3)[k % 3] * (1 + k % 5)), dtype=np.uint8) for k in range(n)]
    bufs = [torch.from_numpy(h).to(device) for h in host]
    vpa.copy_blocks(bufs, u32([1, 4], device), u32([5, 2], device))
    for h, b in zip(host, bufs):
        h[5], h[2] = h[1], h[4]
        assert np.array_equal(b.cpu().numpy(), h)


def test_buffers_looked_at_once(device):
    """BlockBuffers in place of the tensors: the same copies, and refused for another pool."""
    b = Both(device, 40, 8, 6, 6)
    tensors = b.buffers
    once = vpa.BlockBuffers(tensors)
    b.shuffle()
    b.allocate([21, 30, 0, 0, 0, 0])
    b.buffers = once
    b.fork([0, 1, 0], [2, 3, 4])
    b.release([99, 0, 99, 99, 99, 99])
    b.trim([21, 0, 10, 30, 21, 0])
    b.compact()
    b.buffers = tensors
    b.check()
    vpa.copy_blocks(once, u32([1], device), u32([39], device))
    assert all(torch.equal(t[1], t[39]) for t in tensors)
    with pytest.raises(vpa.VpaError, match="40 blocks"):
        vpa.DeviceBlockAllocator(41, 8, 2, 2, device).compact(once)
    for bad, match in (([], "empty"), ([torch.zeros(3)], "GPU only"),
                       ([tensors[0], torch.zeros((41, 2), device=device)], "pools of 40")):
        with pytest.raises(vpa.VpaError, match=match):
            vpa.BlockBuffers(bad)


def test_refusals(device):
    a = vpa.DeviceBlockAllocator(10, 16, 4, 3, device)
    b = torch.zeros((10, 4), device=device)
    with pytest.raises(vpa.VpaError, match="u32 1-d"):
        a.fork(torch.zeros(2, dtype=torch.int64, device=device), u32([1, 2], device), [b])
    with pytest.raises(vpa.VpaError, match="pools of 10"):
        a.fork(u32([0], device), u32([1], device), [torch.zeros((9, 4), device=device)])
    with pytest.raises(vpa.VpaError, match="1024"):
        a.fork(u32(np.zeros(1025), device), u32(np.zeros(1025), device), [b])
    with pytest.raises(vpa.VpaError, match="contiguous blocks"):
        vpa.copy_blocks([torch.zeros((10, 4, 4), device=device)[:, :, :2]], u32([0], device),
                        u32([1], device))
    with pytest.raises(vpa.VpaError, match="GPU only"):
        a.compact([torch.zeros(10, 4)])
    with pytest.raises(vpa.VpaError, match="num_pairs"):
        vpa.copy_blocks([b], u32([0], device), u32([1], device), u32([1, 2], device))
