"""GPU tests of paged_attention_weights over the rows of whole prompts (more than 16 per kv
head): the workspace such a call needs, no more and no less, and the scores against the
64-bit restatement. Bounds as in the tests of the weights."""

import numpy as np
import pytest
import torch

import vpa
from tests._util import u32
from tests.test_gpu_weights import U, check, problem

pytestmark = pytest.mark.gpu


def call(device, p, scores, ws=None):
    rows = np.diff(p["cu"].astype(int))
    return vpa.paged_attention_weights(
        p["q"], p["kc"], p["ks"], u32(p["tables"], device), u32(p["lens"], device), p["d"] ** -0.5,
        scores, cu_seqlens_q=u32(p["cu"], device), max_query_len=int(rows.max()),
        max_context_len=int(p["lens"].max()), workspace=ws)


@pytest.mark.parametrize("dtype,fp8,d,bs,h,kvh", [
    (torch.bfloat16, False, 128, 16, 4, 2), (torch.float16, True, 64, 32, 2, 2),
    (torch.float32, False, 96, 8, 3, 1), (torch.float32, True, 64, 16, 4, 4)])
@pytest.mark.parametrize("lens,rows", [([700, 300, 5], [700, 300, 5]), ([1100, 260], [400, 17]),
                                       ([33], [33])])
def test_exact_workspace(device, dtype, fp8, d, bs, h, kvh, lens, rows):
    """The bytes of the size query, with a guard behind them that stays."""
    p = problem(device, dtype, fp8, d, bs, h, kvh, lens, rows=rows, seed=d + len(lens))
    need = vpa.paged_attention_weights_workspace(sum(rows), h, max(lens), device,
                                                 max_query_len=max(rows), num_kv_heads=kvh).numel()
    buf = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device=device)
    got = call(device, p, p["scores"].clone(), buf[:need])
    check(p, got)
    assert (buf[need:] == 0xA5).all()
    assert torch.equal(got, call(device, p, p["scores"].clone()))
    with pytest.raises(vpa.VpaError, match="bytes needed"):
        call(device, p, p["scores"].clone(), buf[:need - 8])


def test_a_call_allocates_what_it_uses(device):
    """4000 rows of 16 heads over 4000 tokens: 8 MB of pairs (logits would take 1 GB)."""
    n = 4000
    p = problem(device, torch.bfloat16, False, 64, 16, 16, 8, [n], rows=[n], seed=2)
    scores = torch.zeros((1, 8, p["scores"].shape[2]), device=device)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    call(device, p, scores)
    assert torch.cuda.max_memory_allocated() - before < 16 << 20
    # every row's weights sum to 1
    size = 64 ** -0.5 * float(p["q"].float().abs().sum(-1).max()) * float(p["kc"].float().abs().max())
    rel = (2 * 67 * size + 24 + 2 * size + 2 * n + 2) * U
    total = scores.double().sum(-1)
    assert torch.all((total - 2 * n).abs() <= 2 * n * rel)
    assert not scores[..., n:].any()
