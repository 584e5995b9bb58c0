"""GPU tests of what a row of a prompt must not take from tokens that it does not see: the
value scales of later blocks, however far they are from those it sees."""

import numpy as np
import pytest
import torch

from tests import _serving_oracle as ref
from tests.test_gpu_block_scaled import TYPES, UNIT, Problem

pytestmark = pytest.mark.gpu


def louder(p, s, first, last, exponent):
    """Value scales of blocks first .. last - 1 of sequence s, 2^exponent of what they were."""
    ids = p.tables[s, :-(-int(p.lens[s]) // p.bs)][first:last]
    p.vs[ids] = np.ldexp(p.vs[ids], exponent).astype(np.float32)


@pytest.mark.parametrize("d,bs", [(64, 8), (96, 16), (128, 8), (128, 16), (128, 32), (192, 16), (256, 8),
                                  (256, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("exponent", [8, 16, 22, 33, 100])
def test_louder_blocks_that_rows_do_not_see(device, dtype, d, bs, exponent):
    """A quiet block, then one far louder inside the same steps of keys: rows that end in the
    quiet one are as exact as without it, the others as their own scales allow."""
    p = Problem(device, d + bs + exponent, dtype, 4, 2, d, bs, [40, 20, 100], rows=[40, 10, 77])
    p.vs = np.ldexp(p.vs, -40).astype(np.float32)
    for s, first in ((0, 1), (1, -(-20 // bs) - 1), (2, 3)):
        louder(p, s, first, None, exponent)
    p.check()


def test_louder_blocks_of_16_bit_outputs(device):
    """f16 results, whose range holds both."""
    for bs in (8, 16):
        p = Problem(device, bs, torch.float16, 4, 2, 128, bs, [60, 33], rows=[60, 33], spread=1)
        p.vs[:] = 2.0 ** -11
        louder(p, 0, 1, None, 16)
        louder(p, 1, 2, None, 16)
        p.check()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows", [[200], [31], [18]])
def test_a_row_s_result_stands_whatever_later_scales_are(device, dtype, rows):
    """The same rows, with the scales of blocks behind them replaced by anything finite: within
    the bound of the unchanged problem."""
    p = Problem(device, 21, dtype, 4, 2, 64, 8, [200], rows=rows)
    want, *rest = ref.attention(p.q.float().numpy(), p.ks, p.vs, p.kc, p.vc, p.tables, p.lens, p.scale,
                                p.cu)
    bound = ref.attention_bound(want, *rest, 64, 200, UNIT[dtype])
    block = (200 - (rows[0] + 1) // 2) // 8
    seen = block * 8 - (200 - rows[0])  # rows that end before the changed blocks
    assert seen > 0
    for exponent in (0, -60, 5, 30, 119):
        q = Problem(device, 21, dtype, 4, 2, 64, 8, [200], rows=rows)
        louder(q, 0, block, None, exponent)
        got = q.run().float().cpu().numpy().astype(np.float64)
        err = np.abs(got - want)[:seen]
        assert np.all(err <= bound[:seen]), (exponent, np.max(err / bound[:seen]))


def test_loud_blocks_with_no_weight(device):
    """Visible blocks of 2^30 louder values whose probabilities are as much smaller."""
    for rows in (None, [90]):
        p = Problem(device, 23, torch.float32, 2, 1, 64, 16, [90], rows=rows)
        louder(p, 0, 2, 4, 30)
        # 20 nats below the others
        p.q[:] = 1.0
        p.kc[p.tables[0, 2:4]] = 0xB8  # -1
        p.ks[p.tables[0, 2:4]] = 20.0 / (64 * p.scale)
        p.check()


def test_odd_and_negative_scales_apart(device):
    for rows in (None, [120, 64]):
        for dtype in (torch.bfloat16, torch.float32):
            p = Problem(device, 24, dtype, 4, 2, 128, 8, [120, 64], rows=rows, any_scale=True)
            p.vs[p.tables[0, 1::2]] *= np.float32(-(2.0 ** 23))
            louder(p, 1, 3, 5, -70)
            p.check()


@pytest.mark.parametrize("bs", [8, 16, 32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_small_probabilities_beside_a_block_somewhat_louder(device, dtype, bs):
    """Rows whose result is made of probabilities of 2^-28: they count by the scale that the
    rows see, not by that of the next block, 24 times as large."""
    p = Problem(device, 31, dtype, 2, 1, 64, bs, [2 * bs], rows=[2 * bs])
    first, second = p.tables[0, :2]
    p.q[:] = 1.0
    p.kc[:] = 0xB8  # -1
    p.kc[first, :, :, 0] = 0x38  # 1: the first token, the others 28.5 bits below it
    p.ks[:] = 28.5 * np.log(2) / 2 / (64 * p.scale)
    p.vc[:] = 0x7E  # 448, of the first token 0
    p.vc[first, :, :, 0] = 0
    p.vs[first], p.vs[second] = 1.0, 24.0
    got = p.check()
    assert (got[1:bs] > 0).all()


@pytest.mark.parametrize("seed", range(6))
def test_prompts_over_scales_of_any_size(device, seed):
    """Random scales of 2^-48 to 2^40 times odd numbers: every row by the largest that it sees,
    beside rows that see a block or two more."""
    rng = np.random.default_rng(seed)
    lens, rows = rng.integers(0, 71, size=40), rng.integers(0, 90, size=40)
    p = Problem(device, seed, torch.float32, 14, 2, 96, (8, 16)[seed % 2], lens, rows=rows,
                any_scale=seed > 2, spread=20)
    p.vs *= np.ldexp(1.0, rng.integers(-40, 41, size=p.vs.shape)).astype(np.float32)
    p.check()
