"""GPU tests of adjust_logits against a 64-bit model. Each step is one f32 operation:
the result is within 6 * 2^-24 of the largest magnitude it went through, and half a step of
the logits' type (16 bits: a whole one where that error reaches a tie)."""

import numpy as np
import pytest
import torch

import vpa
from tests import _serving_oracle as ref
from tests._util import u32

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


class Case:
    def __init__(self, device, seed, dtype, b, v, k=0, gen=40, prompt=60, bias=5, masks=2,
                 repeat=True, offset=0, wide=0):
        rng = np.random.default_rng(seed)
        self.device, self.dtype, self.b, self.k, self.v = device, dtype, b, k, v
        span = max(1, v // 20) if repeat else v
        flat = torch.from_numpy(rng.standard_normal(offset + b * (k + 1) * (v + wide)).astype(
            np.float32) * 3).to(dtype).to(device)
        self.logits = flat[offset:].view(b, k + 1, v + wide)[..., :v]
        self.outside = flat
        self.x = self.logits.float().cpu().numpy().astype(np.float64)
        ids = lambda n: rng.integers(0, span, size=(b, n)).astype(np.uint32)  # noqa: E731
        self.gen, self.gen_len = ids(gen), rng.integers(0, gen + 3, size=b).astype(np.uint32)
        self.prompt = ids(prompt) if prompt else None
        self.prompt_len = rng.integers(0, prompt + 1, size=b).astype(np.uint32) if prompt else None
        self.drafts = ids(k) if k else None
        self.rep, self.pres, self.freq = (rng.uniform(a, c, size=b).astype(np.float32)
                                          for a, c in ((0.8, 1.5), (-0.5, 1.0), (-0.2, 0.8)))
        self.bias_ids = ids(bias) if bias else None
        self.bias = rng.uniform(-9, 9, size=(b, bias)).astype(np.float32) if bias else None
        self.bias_len = rng.integers(0, bias + 1, size=b).astype(np.uint32) if bias else None
        words = -(-v // 32)
        self.masks = rng.integers(0, 1 << 32, size=(masks, words + 1), dtype=np.uint64).astype(
            np.uint32) if masks else None
        self.which = rng.integers(0, masks + 1, size=(b, k + 1)).astype(np.uint32) if masks else None

    def run(self, **over):
        t = lambda a: None if a is None else (  # noqa: E731
            u32(a, self.device) if a.dtype == np.uint32 else torch.from_numpy(a).to(self.device))
        args = dict(prompt=t(self.prompt), prompt_len=t(self.prompt_len), draft_ids=t(self.drafts),
                    repetition=t(self.rep), presence=t(self.pres), frequency=t(self.freq),
                    bias_ids=t(self.bias_ids), bias=t(self.bias), bias_len=t(self.bias_len),
                    allowed=t(self.masks), allowed_rows=t(self.which))
        args.update(over)
        got = vpa.adjust_logits(self.logits, t(self.gen), t(self.gen_len), **args)
        assert got is self.logits
        torch.cuda.synchronize()
        return got.float().cpu().numpy().astype(np.float64)

    def want(self, b, i):
        told = list(self.gen[b, :min(int(self.gen_len[b]), self.gen.shape[1])])
        if self.drafts is not None:
            told += list(self.drafts[b, :i])
        asked = [] if self.prompt is None else self.prompt[b, :self.prompt_len[b]]
        bias = [] if self.bias is None else list(zip(self.bias_ids[b], self.bias[b]))[:self.bias_len[b]]
        mask = None
        if self.masks is not None and self.which[b, i] < len(self.masks):
            row = self.masks[self.which[b, i]]
            mask = np.unpackbits(row.view(np.uint8), bitorder="little")[:self.v].astype(bool)
        if self.rep is None:
            return ref.adjust(self.x[b, i], told if self.pres is not None else [], bias=bias, mask=mask)
        return ref.adjust(self.x[b, i], told, asked, float(self.rep[b]), float(self.pres[b]),
                          float(self.freq[b]), bias, mask)

    def check(self, **over):
        got = self.run(**over)
        for b in range(self.b):
            for i in range(self.k + 1):
                want, mag = self.want(b, i)
                g = got[b, i]
                nan = np.isnan(want)
                assert np.array_equal(np.isnan(g), nan)
                inf = np.isinf(want)
                assert np.array_equal(g[inf], want[inf])
                fine = ~(nan | inf)
                err = np.abs(g[fine] - want[fine])
                bound = (6 * 2.0 ** -24 * mag + 2 * UNIT[self.dtype] * np.abs(want))[fine]
                same = (mag == np.abs(self.x[b, i]))[fine] & (want == self.x[b, i])[fine]
                assert np.all(err[same] == 0), "an untouched logit changed"
                assert np.all(err <= bound + LEAST[self.dtype]), (b, i, np.max(err / np.maximum(bound, 1e-30)))
        return got


@pytest.mark.parametrize("dtype", list(UNIT), ids=str)
@pytest.mark.parametrize("v", [1, 7, 31, 32, 33, 1000, 16384, 16392, 40001])
def test_sizes(device, dtype, v):
    Case(device, v, dtype, 3, v).check()


@pytest.mark.parametrize("dtype", list(UNIT), ids=str)
@pytest.mark.parametrize("k", [1, 4])
def test_drafted_rows(device, dtype, k):
    Case(device, k, dtype, 4, 501, k=k, gen=12).check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("offset,wide", [(1, 0), (3, 5), (4, 16), (8, 1)])
def test_rows_off_their_alignment(device, dtype, offset, wide):
    """Rows that start and end anywhere; what lies between them stays."""
    c = Case(device, offset, dtype, 3, 997, k=1, offset=offset, wide=wide)
    before = c.outside.clone()
    c.check()
    after = c.outside
    if wide:
        gap = lambda t: t[offset:].view(3, 2, 997 + wide)[..., 997:]  # noqa: E731
        assert torch.equal(gap(before), gap(after))
    assert torch.equal(before[:offset], after[:offset])


@pytest.mark.parametrize("gen,prompt", [(3000, 0), (9000, 2), (5, 20000), (14000, 14000)])
def test_long_lists(device, gen, prompt):
    """Up to 12288 listed tokens are counted in a hash table, more over the vocabulary."""
    for repeat in (True, False):
        Case(device, gen, torch.bfloat16, 2, 70000, k=1, gen=gen, prompt=prompt, repeat=repeat).check()


def test_every_token_of_a_full_table(device):
    """A row that lists as many different tokens as it can."""
    c = Case(device, 5, torch.float32, 2, 30000, gen=12000, prompt=0, bias=200)
    c.gen[:] = np.random.default_rng(1).permutation(30000)[:12000].astype(np.uint32)
    c.gen_len[:] = 12000
    c.check()


def test_each_part_alone(device):
    none = dict(repetition=None, presence=None, frequency=None)
    for bias, masks in ((5, 0), (0, 2), (0, 0), (5, 2)):
        c = Case(device, bias + masks, torch.bfloat16, 3, 777, bias=bias, masks=masks)
        c.rep = c.pres = c.freq = None
        c.check(**none)
    c = Case(device, 1, torch.float32, 3, 777, bias=0, masks=0)
    c.rep[:], c.freq[:] = 1.0, 0.0
    c.check(repetition=None, frequency=None, prompt=None, prompt_len=None)
    c = Case(device, 2, torch.float32, 3, 777, bias=0, masks=0)
    c.pres[:], c.freq[:] = 0.0, 0.0
    c.check(presence=None, frequency=None)


def test_ids_past_the_vocabulary_and_lengths_past_the_list(device):
    c = Case(device, 4, torch.float32, 3, 100, gen=20, prompt=9, bias=6)
    for a in (c.gen, c.prompt, c.bias_ids):
        a[:, ::2] += np.uint32(95)
        a[0, 1] = 0xFFFFFFFF
    c.gen_len[:] = [0xFFFFFFFF, 0, 21]
    c.bias_len[:] = 6
    c.check()
    # no lengths: the whole lists
    c = Case(device, 5, torch.float32, 3, 100, gen=20, prompt=9, bias=6)
    c.gen_len[:], c.prompt_len[:], c.bias_len[:] = 20, 9, 6
    got = c.run(prompt_len=None, bias_len=None)
    for b in range(3):
        want, mag = c.want(b, 0)
        fine = np.isfinite(want)
        assert np.all(np.abs(got[b, 0][fine] - want[fine]) <= (8 * 2.0 ** -24 * mag)[fine] + 1e-40)


def test_last_of_equal_biases_counts(device):
    c = Case(device, 6, torch.float32, 2, 64, bias=40, masks=0)
    c.bias_ids[:] = c.bias_ids % 5
    c.bias_len[:] = [40, 17]
    c.check()


def test_special_logits(device):
    """-inf and NaN go through; zeros are not positive; a bias of -inf bans a token."""
    c = Case(device, 7, torch.float32, 2, 64, gen=10, masks=1)
    c.logits[0, 0, :4] = torch.tensor([-np.inf, np.nan, 0.0, -0.0], device=device)
    c.x = c.logits.cpu().numpy().astype(np.float64)
    c.gen[0, :4], c.gen_len[0] = [0, 1, 2, 3], 10
    c.bias_ids[1, 0], c.bias[1, 0], c.bias_len[1] = 9, -np.inf, 1
    c.check()


def test_masks(device):
    """Nothing allowed, all allowed, one token in each place of a vector; a mask per row
    without allowed_rows; stray bits behind the vocabulary."""
    v = 203
    for dtype in UNIT:
        c = Case(device, 8, dtype, 40, v, gen=3, prompt=0, bias=0, masks=40)
        c.masks[:] = 0
        c.masks[1] = 0xFFFFFFFF
        for i in range(2, 40):
            at = 5 * i + 1
            c.masks[i, at // 32] = 1 << (at % 32)
            c.masks[i, -1] = 0xFFFFFFFF
        c.which = np.arange(40, dtype=np.uint32)[:, None]
        c.check(allowed_rows=None)


def test_two_dimensional_logits_and_a_slice(device):
    x = torch.randn((6, 300), device=device)
    gen, n = u32(np.full((3, 2), 7), device), u32([2, 0, 1], device)
    rep = torch.full((3,), 2.0, device=device)
    want = x.clone()
    for r, k in ((0, 1), (4, 1)):
        want[r, 7] = want[r, 7] / 2 if want[r, 7] > 0 else want[r, 7] * 2
    vpa.adjust_logits(x[::2], gen, n, repetition=rep)
    assert torch.equal(x, want)


def test_refusals(device):
    x = torch.zeros((2, 3, 40), device=device)
    ok = u32(np.zeros((2, 4)), device)
    f = torch.ones(2, device=device)
    for bad, needle in (
            (dict(generated=ok.view(torch.int32)), "generated"),
            (dict(generated=ok[:1]), "generated"), (dict(generated=ok, gen_len=ok[0]), "lengths"),
            (dict(gen_len=ok[:, 0]), "without"), (dict(draft_ids=ok), "draft_ids"),
            (dict(repetition=f.double()), "repetition"), (dict(presence=f[:1]), "presence"),
            (dict(bias_ids=ok), "bias"), (dict(bias=torch.zeros(2, 4, device=device)), "bias"),
            (dict(allowed=ok), "num_masks"), (dict(allowed=ok.view(torch.int32)), "allowed"),
            (dict(allowed_rows=ok), "without"), (dict(allowed=ok, allowed_rows=ok), "allowed_rows"),
            (dict(allowed=ok[:, :1], allowed_rows=u32(np.zeros((2, 3)), device)), "allowed_stride")):
        with pytest.raises(vpa.VpaError, match=needle):
            vpa.adjust_logits(x, **bad)
    with pytest.raises(vpa.VpaError, match="contiguous"):
        vpa.adjust_logits(torch.zeros((2, 40, 2), device=device).transpose(1, 2))
    with pytest.raises(vpa.VpaError, match="overlap"):
        vpa.adjust_logits(torch.zeros((1, 40), device=device).expand(3, 40))
    with pytest.raises(vpa.VpaError, match="GPU only"):
        vpa.adjust_logits(torch.zeros(2, 40))
    assert not x.any()
