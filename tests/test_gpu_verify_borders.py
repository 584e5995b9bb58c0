"""GPU tests of verify_draft_tokens right at the borders of its decisions. The weights are f64
within 4e-14 and 3 half units of their exponents (below 1e-13 at the logits here), and a
sum adds about a hundred additions of 2^-53 each: a decision is certain where the exact one
is farther than 5e-13 (relatively) from its border. The exact values are 80-bit."""

import numpy as np
import pytest
import torch

import vpa

pytestmark = pytest.mark.gpu

CLEAR = 5e-13


def weights(row, temp):
    row = row.astype(np.longdouble)
    return np.exp((row - row.max()) / np.longdouble(temp))


@pytest.mark.parametrize("spread,temp", [(0.01, 1.0), (2.5, 0.7)])
def test_draws_of_a_large_vocabulary(device, spread, temp):
    """4000 draws from one row of 100 003 tokens (a zero stride), each exact."""
    gen = torch.Generator().manual_seed(1)
    b, v = 4000, 100003
    row = spread * torch.randn(v, generator=gen)
    u = torch.rand(b, generator=gen)
    temps = torch.full((b,), temp)
    up = np.cumsum(weights(row.numpy(), float(temps[0])))
    target = u.numpy().astype(np.longdouble) * up[-1]
    want = np.searchsorted(up, target, side="right")
    near = np.minimum(np.abs(up[want] - target), np.abs(up[np.maximum(want - 1, 0)] - target))
    clear = near > CLEAR * up[-1]
    assert clear.mean() > 0.999
    got, count = vpa.verify_draft_tokens(
        row.to(device).expand(b, 1, v), torch.zeros((b, 0), dtype=torch.uint32, device=device),
        torch.zeros((b, 0), device=device), u.to(device), temperature=temps.to(device))
    assert (count.cpu().numpy() == 1).all()
    assert np.array_equal(got.cpu().numpy()[clear, 0], want[clear])


@pytest.mark.parametrize("looked_up", [False, True])
def test_acceptance_between_neighbouring_numbers(device, looked_up):
    """Each draft with the f32 accept_u just below and just above its exact border p / q."""
    gen = torch.Generator().manual_seed(2)
    b, v = 200, 4999
    target = 2 * torch.randn((b, 2, v), generator=gen)
    draft = target[:, :1] + torch.randn((b, 1, v), generator=gen)
    temp = 0.5 + torch.rand(b, generator=gen)
    ids = draft[:, 0].argmax(-1) if not looked_up else target[:, 0].argmax(-1)
    border = np.empty(b, np.longdouble)
    for s in range(b):
        p, x = weights(target[s, 0].numpy(), float(temp[s])), int(ids[s])
        border[s] = p[x] / p.sum()
        if not looked_up:
            q = weights(draft[s, 0].numpy(), float(temp[s]))
            border[s] *= q.sum() / q[x]
    low = border.astype(np.float32)
    low = np.where(low.astype(np.longdouble) < border, low, np.nextafter(low, np.float32(0)))
    use = border < 1
    assert use.sum() > b // 4
    tried = 0
    for u, accepted in ((low, True), (np.nextafter(low, np.float32(2)), False)):
        certain = use & (np.abs(u.astype(np.longdouble) / border - 1) > CLEAR) & (u < 1)
        got, count = vpa.verify_draft_tokens(
            target.to(device), ids[:, None].to(torch.int32).view(torch.uint32).to(device),
            torch.from_numpy(u)[:, None].to(device), torch.full((b,), 0.5, device=device),
            draft_logits=None if looked_up else draft.to(device), temperature=temp.to(device))
        assert np.array_equal(count.cpu().numpy()[certain] == 2, np.full(int(certain.sum()), accepted))
        tried += int(certain.sum())
    assert tried > use.sum()
