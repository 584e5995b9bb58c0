"""GPU tests of shared blocks that a row is about to write to: every one behind its tokens is
replaced, whatever it was set back to."""

import numpy as np
import pytest
import torch

import vpa
from tests._util import u32
from vpa import _lib

pytestmark = pytest.mark.gpu

BS, NB, ROWS, COLS = 8, 40, 6, 6


class Rows:
    """An allocator with its state on the host, taken one row and block at a time."""

    def __init__(self, device, tokens):
        self.device = device
        self.dev = vpa.DeviceBlockAllocator(NB, BS, ROWS, COLS, device)
        self.pool = torch.arange(NB * 4, device=device, dtype=torch.float32).view(NB, 4)
        self.dev.enable_sharing()
        self.dev.allocate(u32(tokens, device))
        self.dev.positions.copy_(u32(tokens, device))

    def fork(self, src, dst):
        assert self.dev.fork(u32(src, self.device), u32(dst, self.device), [self.pool]).cpu().all()

    def state(self):
        torch.cuda.synchronize()
        d = self.dev
        return {n: getattr(d, n).cpu().numpy().copy() for n in (
            "block_tables", "row_blocks", "positions", "shared", "free_ring", "free_ring_state")}

    def unshare(self):
        """The entry point alone: (ok, pairs)."""
        d = self.dev
        ok = torch.full((ROWS,), 9, dtype=torch.uint8, device=self.device)
        src, dst = (u32(np.full(ROWS, 77), self.device) for _ in range(2))
        count = u32([99], self.device)
        rc = _lib.load().vpa_unshare_rows(
            d.block_tables.data_ptr(), COLS, d.row_blocks.data_ptr(), d.positions.data_ptr(),
            d.shared.data_ptr(), NB, ok.data_ptr(), src.data_ptr(), dst.data_ptr(), count.data_ptr(),
            d.free_ring.data_ptr(), d.free_ring_state.data_ptr(), NB, BS, ROWS,
            torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        n = int(count.cpu()[0])
        return ok.cpu().numpy(), list(zip(src.cpu().tolist()[:n], dst.cpu().tolist()[:n]))


def unshared(s):
    """What unshare_rows makes of a state: (state, ok, pairs)."""
    s = {k: v.copy() for k, v in s.items()}
    ok, pairs = np.ones(ROWS, np.uint8), []
    head, avail = (int(x) for x in s["free_ring_state"])
    for r in range(ROWS):
        at, inside = divmod(int(s["positions"][r]), BS)
        for i in range(at, min(int(s["row_blocks"][r]), COLS)):
            b = int(s["block_tables"][r, i])
            if b == 0 or b >= NB or s["shared"][b] == 0:
                continue
            if avail == 0:
                ok[r] = 0
                continue
            new = int(s["free_ring"][head])
            head, avail = (head + 1) % NB, avail - 1
            s["shared"][b] -= 1
            s["block_tables"][r, i] = new
            if i == at and inside:
                pairs.append((b, new))
    s["free_ring_state"][:] = head, avail
    return s, ok, pairs


def same(a, b):
    for k in a:
        assert np.array_equal(a[k], b[k]), k


@pytest.mark.parametrize("cut", [24, 17, 16, 11, 8, 3, 0])
@pytest.mark.parametrize("both", [False, True])
def test_rows_set_back_without_a_release(device, cut, both):
    """Positions alone were set back, to a block's start, inside one, over several: every
    shared block that the row would write to is its own afterwards."""
    b = Rows(device, [29, 0, 0, 10, 0, 0])
    b.fork([0, 0], [1, 2])
    at = [cut if both else 29, cut, 29, 10, 0, 0]
    b.dev.positions.copy_(u32(at, device))
    want, ok, pairs = unshared(b.state())
    got_ok, got_pairs = b.unshare()
    same(b.state(), want)
    assert got_ok.tolist() == ok.tolist() and got_pairs == pairs
    # nobody's next token falls into a block that others hold
    s = b.state()
    for r in range(ROWS):
        for i in range(at[r] // BS, int(s["row_blocks"][r])):
            assert s["shared"][s["block_tables"][r, i]] == 0


def test_random_rows_set_back(device):
    rng = np.random.default_rng(3)
    for _ in range(12):
        b = Rows(device, [int(rng.integers(0, COLS * BS)), int(rng.integers(0, 20)), 0, 0, 0, 0])
        b.fork([0, 1, 0], [2, 3, 4])
        s = b.state()
        b.dev.positions.copy_(u32((s["positions"] * rng.random(ROWS)).astype(np.uint32), device))
        if rng.random() < 0.5:  # few blocks left
            s["free_ring_state"][1] = rng.integers(0, 4)
            b.dev.free_ring_state.copy_(u32(s["free_ring_state"], device))
        want, ok, pairs = unshared(b.state())
        got_ok, got_pairs = b.unshare()
        same(b.state(), want)
        assert got_ok.tolist() == ok.tolist() and got_pairs == pairs
