"""Refusals of DeviceBlockAllocator.release before its entry point reads keep_blocks (no GPU here)."""

import pytest
import torch

import vpa


@pytest.mark.parametrize("sharing", [False, True])
@pytest.mark.parametrize("keep,needle", [
    (torch.zeros(3, dtype=torch.uint32), "u32"), (torch.zeros((4, 1), dtype=torch.uint32), "u32"),
    (torch.zeros(4, dtype=torch.int64), "u32"), (torch.zeros(4), "u32"),
    (torch.zeros(8, dtype=torch.uint32)[::2], "GPU only")])
def test_keep_blocks(sharing, keep, needle):
    a = vpa.DeviceBlockAllocator(10, 16, 4, 3, "cpu")
    if sharing:
        a.enable_sharing()
    with pytest.raises(vpa.VpaError, match=needle):
        a.release(keep)
