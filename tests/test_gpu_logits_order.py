"""GPU test of logits whose draft rows lie outside their sequences, [K + 1, B, V] in memory."""

import pytest
import torch

import vpa
from tests._util import u32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_drafts_slowest_in_memory(device, dtype):
    gen = torch.Generator().manual_seed(1)
    b, k1, v = 3, 4, 130
    x = torch.randn((k1, b, v), generator=gen).to(dtype).to(device)
    ids = torch.randint(0, v, (b, 20), generator=gen).int().to(device).view(torch.uint32)
    drafts = torch.randint(0, v, (b, k1 - 1), generator=gen).int().to(device).view(torch.uint32)
    rep = torch.full((b,), 1.7, device=device)
    want = x.transpose(0, 1).contiguous()
    vpa.adjust_logits(want, ids, draft_ids=drafts, repetition=rep)
    got = x.transpose(0, 1)
    assert vpa.adjust_logits(got, ids, draft_ids=drafts, repetition=rep) is got
    assert torch.equal(got.contiguous(), want)


def test_overlapping_rows_are_refused(device):
    x = torch.zeros(4000, device=device)
    one = u32([[1], [1]], device)
    rep = torch.ones(2, device=device)
    for strides in ((150, 100, 1), (100, 150, 1), (50, 300, 1), (0, 300, 1)):
        with pytest.raises(vpa.VpaError, match="overlap"):
            vpa.adjust_logits(x.as_strided((2, 3, 100), strides), one, repetition=rep)
