"""GPU tests of NaN bytes of V in steps of keys that every row sees but for an absent block."""

import numpy as np
import pytest
import torch

from tests.test_gpu_block_scaled import Problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bs", [8, 16])
@pytest.mark.parametrize("rows", [None, [30], [150]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_nan_beside_an_absent_block(device, dtype, rows, bs):
    """A NaN of V in a step of keys that every row sees whole, with an absent block in it."""
    p = Problem(device, 25, dtype, 2, 1, 64, bs, [300], rows=rows)
    p.tables[0, 1] = 0xFFFFFFFF
    at = 2 * bs + 3
    p.vc[p.tables[0, at // bs], 0, 9, at % bs] = 0x7F
    got = p.check()
    assert np.isnan(got[..., 9]).all() and not np.isnan(np.delete(got, 9, axis=-1)).any()


def test_nan_beside_an_absent_block_stays_with_its_rows(device):
    """One in the middle of a prompt's rows: those before it have none."""
    p = Problem(device, 26, torch.bfloat16, 2, 1, 64, 16, [200], rows=[200])
    p.tables[0, 5] = 5000
    at = 100
    p.vc[p.tables[0, at // 16], 0, 7, at % 16] = 0xFF
    got = p.check()
    assert np.isnan(got[at:, :, 7]).all() and not np.isnan(got[:at]).any()
