"""GPU tests of rows that share the block they would write to next and found no block of their
own: they do not run, so that nobody else's block is written, and go on once they can."""

import pytest
import torch

import vpa
from tests._util import u32
from tests.test_gpu_pages_unshare import BS, COLS, NB, ROWS, Rows, same

pytestmark = pytest.mark.gpu


def full_pool(device):
    """Rows 0 and 1 cut back to inside a block that they and row 2 hold, none left."""
    b = Rows(device, [24, 0, 0, 0, 0, 0])
    b.fork([0, 0], [1, 2])
    state = b.dev.free_ring_state.cpu().numpy()
    b.dev.free_ring_state.copy_(u32([state[0], 0], device))
    b.dev.trim(u32([20, 21, 24, 0, 0, 0], device), buffers=[b.pool])
    assert b.dev.ok.cpu().tolist() == [0, 0, 1, 1, 1, 1]
    return b, state


def test_a_row_without_a_block_of_its_own_does_not_run(device):
    b, state = full_pool(device)
    finished = torch.tensor([0, 0, 1, 1, 1, 1], dtype=torch.uint8, device=device)
    for _ in range(2):
        before = b.state()
        slots, lens = b.dev.step(finished)
        assert (slots.cpu().numpy() < 0).all() and (lens.cpu().numpy() == 1).all()
        assert b.dev.status.cpu().tolist()[:2] == [2, 0]  # both stalled
        same(b.state(), before)
    # with blocks again, a trim gives each its own; they go on where they stood
    b.dev.free_ring_state.copy_(u32(state, device))
    b.dev.trim(u32([20, 21, 24, 0, 0, 0], device), buffers=[b.pool])
    assert b.dev.ok.cpu().all()
    s = b.state()
    held = [int(s["block_tables"][r, 2]) for r in range(3)]
    assert len(set(held)) == 3 and all(s["shared"][x] == 0 for x in held)
    slots, lens = b.dev.step(finished)
    assert slots.cpu().tolist()[:2] == [held[0] * BS + 4, held[1] * BS + 5]
    assert lens.cpu().tolist()[:2] == [21, 22]


def test_it_runs_once_the_others_gave_the_block_back(device):
    b, _ = full_pool(device)
    finished = torch.tensor([0, 1, 1, 1, 1, 1], dtype=torch.uint8, device=device)
    block = int(b.state()["block_tables"][0, 2])
    b.dev.release(u32([99, 0, 0, 0, 0, 0], device))
    slots, _ = b.dev.step(finished)
    assert int(slots[0]) == block * BS + 4


def test_a_step_at_a_shared_block_s_start_does_not_run(device):
    """Set back to a block's start without a release or an unshare."""
    b = Rows(device, [24, 0, 0, 0, 0, 0])
    b.fork([0], [1])
    b.dev.positions.copy_(u32([24, 16, 0, 0, 0, 0], device))
    finished = torch.tensor([1, 0, 1, 1, 1, 1], dtype=torch.uint8, device=device)
    slots, _ = b.dev.step(finished)
    assert int(slots[1]) < 0 and b.dev.status.cpu().tolist()[:2] == [1, 0]


def test_rows_of_their_own_step_as_before(device):
    """Forked rows' steps with sharing enabled equal those of the step without shared counts."""
    b = Rows(device, [24, 13, 0, 0, 0, 0])
    b.fork([0, 1, 1], [2, 3, 4])
    plain = vpa.DeviceBlockAllocator(NB, BS, ROWS, COLS, device)
    for n in ("block_tables", "row_blocks", "positions", "free_ring", "free_ring_state"):
        getattr(plain, n).copy_(getattr(b.dev, n))
    finished = torch.tensor([0, 0, 0, 0, 0, 1], dtype=torch.uint8, device=device)
    for _ in range(2 * BS):
        for x, y in zip(b.dev.step(finished), plain.step(finished)):
            assert torch.equal(x.view(torch.int32), y.view(torch.int32))
        assert torch.equal(b.dev.status.view(torch.int32), plain.status.view(torch.int32))
        for n in ("block_tables", "row_blocks", "positions", "free_ring_state"):
            assert torch.equal(getattr(b.dev, n).view(torch.int32), getattr(plain, n).view(torch.int32))


def test_a_stalled_row_s_shared_block_keeps_its_bytes(device):
    """The whole of it: rows of a block-scaled cache, a trim that finds no block, steps of
    append and attention, captured and replayed; what the other holder reads stays."""
    kvh, d, h = 2, 64, 4
    b, _ = full_pool(device)
    kc = torch.randint(0, 120, (NB, kvh, d // 16, BS, 16), dtype=torch.uint8, device=device)
    vc = torch.randint(0, 120, (NB, kvh, d, BS), dtype=torch.uint8, device=device)
    ks, vs = (torch.full((NB, kvh), 2.0 ** -6, device=device) for _ in range(2))
    before = [t.clone() for t in (kc, vc, ks, vs)]
    finished = torch.tensor([0, 0, 1, 1, 1, 1], dtype=torch.uint8, device=device)
    k = 100 * torch.randn((ROWS, kvh, d), device=device)
    q = torch.randn((ROWS, h, d), device=device)
    out = torch.empty_like(q)

    def step():
        slots, lens = b.dev.step(finished)
        vpa.reshape_and_cache_block_scaled(k, k, ks, vs, kc, vc, slots)
        vpa.paged_attention_block_scaled(q, ks, vs, kc, vc, b.dev.block_tables, lens, 0.1,
                                         max_context_len=COLS * BS, out=out)

    step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for t, w in zip((kc, vc, ks, vs), before):
            assert torch.equal(t, w)
