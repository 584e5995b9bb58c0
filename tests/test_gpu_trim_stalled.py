"""GPU tests of DeviceBlockAllocator.trim after a step in which rows did not run: a row that
stalls (no block left for its next token) and a finished one show context_lens 1 and a
negative slot, and go on with all they hold."""

import numpy as np
import pytest
import torch

import vpa
from tests._util import u32

pytestmark = pytest.mark.gpu


def ran_lens(ctx, slots):
    """The step's lengths with 0 for the rows that did not run."""
    return (ctx.view(torch.int32) * (slots >= 0)).view(torch.uint32)


def test_rows_that_did_not_run_keep_their_tokens(device):
    """Row 1 needs a block and gets none; row 3 is finished. The cut of the others to 30
    tokens gives blocks back, and the stalled row goes on where it stood."""
    alloc = vpa.DeviceBlockAllocator(1 + 10, 16, 4, 8, device)
    held = [40, 48, 20, 30]  # 3 + 3 + 2 + 2 blocks: the pool is empty
    assert alloc.allocate(u32(held, device)).all()
    alloc.positions.copy_(u32(held, device))
    tables = alloc.block_tables.cpu().numpy().copy()
    finished = torch.tensor([0, 0, 0, 1], dtype=torch.uint8, device=device)
    slots, ctx = alloc.step(finished)
    assert ctx.cpu().numpy().tolist() == [41, 1, 21, 1]
    assert (slots.cpu().numpy() < 0).tolist() == [False, True, False, True]
    new_lens = u32(np.minimum(ctx.cpu().numpy(), 30), device)
    alloc.trim(new_lens, slots)
    assert alloc.positions.cpu().numpy().tolist() == [30, 48, 21, 30]
    assert alloc.row_blocks.cpu().numpy().tolist() == [2, 3, 2, 2]
    assert int(alloc.free_ring_state[1]) == 1
    slots, ctx = alloc.step(finished)
    assert ctx.cpu().numpy().tolist() == [31, 49, 22, 1]  # (row 0's third block is row 1's now)
    got = alloc.block_tables.cpu().numpy()
    assert np.array_equal(got[1, :3], tables[1, :3]) and got[1, 3] == tables[0, 2]
    assert int(slots[1]) == int(tables[0, 2]) * 16
    with pytest.raises(vpa.VpaError, match="slot_mapping"):
        alloc.trim(new_lens, slots.int())
    with pytest.raises(vpa.VpaError, match="slot_mapping"):
        alloc.trim(new_lens, slots[:3])
    with pytest.raises(vpa.VpaError, match="GPU only"):
        alloc.trim(new_lens, slots.cpu())


def test_weights_eviction_and_trim_with_a_stalled_row(device):
    """The whole cut of a layer in such a step, captured and replayed: the stalled row's
    scores, cache, blocks and length stay as they are."""
    gen = torch.Generator().manual_seed(4)
    rand = lambda *s: torch.randn(s, generator=gen).to(device)  # noqa: E731

    def state():
        alloc = vpa.DeviceBlockAllocator(1 + 6, 16, 2, 6, device)
        assert alloc.allocate(u32([48, 48], device)).all()
        alloc.positions.copy_(u32([47, 48], device))
        return alloc

    q, kc, vc = rand(2, 4, 64), rand(7, 2, 16, 16, 4), rand(7, 2, 64, 16)
    first = rand(2, 2, 96).abs()

    def step(alloc, kc, vc, scores):
        slots, ctx = alloc.step()
        lens = ran_lens(ctx, slots)
        vpa.paged_attention_weights(q, kc, None, alloc.block_tables, lens, 0.125, scores,
                                    max_context_len=96)
        new_lens, _ = vpa.evict_kv_cache(kc, vc, scores, alloc.block_tables, lens, 20, keep_first=2,
                                         keep_last=4, max_context_len=96)
        alloc.trim(new_lens, slots)

    def run_eager():
        a, bufs = state(), [kc.clone(), vc.clone(), first.clone()]
        step(a, *bufs)
        torch.cuda.synchronize()
        return a, bufs

    a, bufs = run_eager()
    assert a.positions.cpu().numpy().tolist() == [20, 48]
    assert a.row_blocks.cpu().numpy().tolist() == [2, 3]
    own = a.block_tables.cpu().numpy()[1, :3].astype(np.int64)
    assert torch.equal(bufs[0][own], kc[own]) and torch.equal(bufs[1][own], vc[own])
    assert torch.equal(bufs[2][1], first[1]) and not torch.equal(bufs[2][0], first[0])
    b, mine = state(), [kc.clone(), vc.clone(), first.clone()]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(b, *mine)
    for _ in range(3):  # (the second step has a block for row 1)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip((*bufs, a.positions, a.row_blocks), (*mine, b.positions, b.row_blocks)):
            x, y = (t.view(torch.int32) if t.dtype == torch.uint32 else t for t in (x, y))
            assert torch.equal(x, y)
        step(a, *bufs)
        torch.cuda.synchronize()
