"""GPU tests of verify_draft_tokens' greedy form (temperature <= 0 or NaN) at its borders:
rows with no number (all -inf or NaN), whose answer is id 0, and drafted ids past the
vocabulary, which are never accepted, the operator's own padding value among them. The
answers are whole numbers and equal those of the 64-bit restatement."""

import numpy as np
import pytest
import torch

import vpa
from tests import _loop_oracle as ref
from tests._util import u32

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")
PAD = 0xFFFFFFFF


def run(device, target, ids, num_drafts=None):
    b, k = ids.shape
    dev = target.to(device)
    return [t.cpu().numpy() for t in vpa.verify_draft_tokens(
        dev, u32(ids, device), torch.zeros((b, k), device=device), torch.zeros(b, device=device),
        num_drafts=None if num_drafts is None else u32(num_drafts, device),
        temperature=torch.zeros(b, device=device))]


def check(device, target, ids, num_drafts=None):
    b, k = ids.shape
    want_ids, want_count, _ = ref.verify(target.double().numpy(), ids, np.zeros((b, k)), np.zeros(b),
                                         None, num_drafts, np.zeros(b))
    got_ids, count = run(device, target, ids, num_drafts)
    assert np.array_equal(count, want_count)
    assert np.array_equal(got_ids, want_ids)
    return got_ids, count


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 5, 4097, 9000])
def test_rows_without_a_number(device, dtype, v):
    """Every row of each kind of nothing, against every kind of draft."""
    drafts = [0, min(5, v), v, v + 1, 2 ** 31, PAD - 1, PAD]
    kinds = [torch.full((v,), -INF), torch.full((v,), NAN),
             torch.where(torch.arange(v) % 2 == 0, NAN, -INF)]
    target = torch.stack([k for k in kinds for _ in drafts])[:, None].repeat(1, 2, 1).to(dtype)
    ids = np.array(drafts * len(kinds), np.uint32)[:, None]
    got, count = check(device, target, ids)
    accepted = ids[:, 0] == 0
    assert (count == 1 + accepted).all() and (got[:, 0] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_numbers_follow_rows_without(device, dtype):
    """Such a row in the middle: an accepted 0 goes on to the row behind it."""
    gen = torch.Generator().manual_seed(1)
    target = torch.randn((4, 4, 700), generator=gen).to(dtype)
    best = target.float().argmax(-1).numpy()
    target[:, 1] = torch.tensor([-INF, NAN, -INF, NAN], dtype=dtype)[:, None]
    ids = best[:, :3].astype(np.uint32)
    ids[:, 1] = [0, 0, PAD, 700]
    got, count = check(device, target, ids)
    assert count.tolist() == [4, 4, 2, 2]
    assert got[0].tolist() == [best[0, 0], 0, best[0, 2], best[0, 3]]


def test_ids_past_the_vocabulary_in_rows_of_numbers(device):
    gen = torch.Generator().manual_seed(2)
    target = torch.randn((5, 3, 4100), generator=gen)
    target[3, 0, 4099] = INF
    ids = target[:, :2].argmax(-1).numpy().astype(np.uint32)
    ids[:3, 0] = [4100, 8191, PAD]
    _, count = check(device, target, ids)
    assert count.tolist() == [1, 1, 1, 3, 3]
    # padded drafts behind num_drafts are not looked at
    ids[4, 1] = PAD
    _, count = check(device, target, ids, np.array([0, 1, 2, 2, 1]))
    assert count.tolist() == [1, 1, 1, 3, 2]
