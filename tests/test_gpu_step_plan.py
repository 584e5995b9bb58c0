"""GPU tests of layers that need the work list of a step that was begun without one."""

import pytest
import torch

import vpa
from tests._util import u32

pytestmark = pytest.mark.gpu

H, KVH, D, BS, NB = 4, 2, 64, 16, 8


def begun(device, block_scaled):
    step = vpa.DeviceDecodeStep(2, NB, BS, 64, H, D, [9], 8, device)
    assert step.admit(u32([5, 20], device)).cpu().all()
    kc = torch.zeros((NB, KVH, D // 16, BS, 16), dtype=torch.uint8, device=device)
    vc = torch.zeros((NB, KVH, D, BS), dtype=torch.uint8, device=device)
    step.begin(kc, vc, torch.float32, block_scaled=block_scaled)
    return step, kc, vc


def layer(step, kc, vc, *scales):
    q, k, v = (torch.ones((2, n, D), device=kc.device) for n in (H, KVH, KVH))
    out = torch.zeros((2, H, D), device=kc.device)
    step.layer(q, k, v, kc, vc, out, *scales)
    return out


def test_a_layer_of_one_scale_in_a_block_scaled_step(device):
    step, kc, vc = begun(device, True)
    one = torch.full((1,), 0.25, device=device)
    with pytest.raises(vpa.VpaError, match="block_scaled"):
        layer(step, kc, vc, one, one)
    assert not kc.any() and not vc.any()  # nothing was appended either
    scales = vpa.block_scales(NB, KVH, device)
    assert layer(step, kc, vc, *scales).any()
    # the next step has a list again
    kc.zero_(), vc.zero_()
    step.begin(kc, vc, torch.float32)
    assert layer(step, kc, vc, one, one).any()


def test_both_kinds_in_a_step_with_a_list(device):
    step, kc, vc = begun(device, False)
    one = torch.full((1,), 0.25, device=device)
    assert layer(step, kc, vc, one, one).any()
    kc.zero_(), vc.zero_()
    assert layer(step, kc, vc, *vpa.block_scales(NB, KVH, device)).any()
