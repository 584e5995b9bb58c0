"""GPU tests of evict_kv_cache over contexts without a token, or with no more than the
budget: the lengths and kept positions are written, the caches and scores stay."""

import numpy as np
import pytest
import torch

import vpa
from tests._util import u32

pytestmark = pytest.mark.gpu


def state(device, b, width):
    gen = torch.Generator().manual_seed(3)
    kc = torch.randn((12, 2, 8, 16, 8), generator=gen).to(device, torch.bfloat16)
    vc = torch.randn((12, 2, 64, 16), generator=gen).to(device, torch.bfloat16)
    return kc, vc, torch.rand((b, 2, width), generator=gen).to(device)


def check(device, lens, budget, width=64, cols=4, **kw):
    b = len(lens)
    kc, vc, sc = state(device, b, width)
    saved = [t.clone() for t in (kc, vc, sc)]
    tables = np.arange(b * cols, dtype=np.uint32).reshape(b, cols) % 12
    new, kept = vpa.evict_kv_cache(kc, vc, sc, u32(tables, device), u32(lens, device), budget, **kw)
    torch.cuda.synchronize()
    assert new.cpu().numpy().tolist() == list(lens)
    for s, n in enumerate(lens):
        want = np.full((2, budget), 0xFFFFFFFF, np.uint32)
        want[:, :n] = np.arange(n)
        assert np.array_equal(kept[s].cpu().numpy(), want)
    assert all(torch.equal(a, b) for a, b in zip(saved, (kc, vc, sc)))


@pytest.mark.parametrize("budget", [1, 40])
@pytest.mark.parametrize("b", [1, 3])
def test_contexts_without_tokens(device, b, budget):
    """max_context_len 0, read from the lengths and given: no workspace is needed."""
    check(device, [0] * b, budget)
    check(device, [0] * b, budget, max_context_len=0, workspace=torch.empty(0, dtype=torch.uint8,
                                                                            device=device))


def test_contexts_within_the_budget(device):
    check(device, [0, 1, 33], 33)
    check(device, [0, 1, 33], 60, keep_first=4, keep_last=9, max_context_len=60)
    check(device, [0, 1, 33], 33, max_context_len=64)


@pytest.mark.parametrize("width,cols", [(0, 4), (64, 0), (0, 0)])
def test_empty_scores_and_tables(device, width, cols):
    """Before the first token scores and tables may have no columns at all (their data
    pointers are null); the weights of such contexts are nothing."""
    check(device, [0, 0], 7, width=width, cols=cols)
    kc, _, sc = state(device, 2, width)
    q = torch.ones((2, 4, 64), dtype=torch.bfloat16, device=device)
    got = vpa.paged_attention_weights(q, kc, None, u32(np.zeros((2, cols)), device), u32([0, 0], device),
                                      1.0, sc)
    assert got is sc and torch.equal(sc, state(device, 2, width)[2])
