"""GPU tests of verify_draft_tokens against the 64-bit restatement: the emitted ids
are whole numbers and equal. Acceptance compares sums of f32 exponentials, each
off by about 2^-22 at the logits used, so a decision may differ only where the exact one
is closer to its border than 2^-20; the tests' fixed inputs are checked to stay
clear of that (the oracle's margins), not adjusted."""

import numpy as np
import pytest
import torch

import vpa
from tests import _loop_oracle as ref

pytestmark = pytest.mark.gpu

MARGIN = 2.0 ** -20


def problem(dtype, b, k, v, *, draft=True, noise=0.7, spread=2.5, seed=0, temps=True, ragged=False,
            greedy=()):
    gen = torch.Generator().manual_seed(seed)
    target = spread * torch.randn((b, k + 1, v), generator=gen)
    dl = (target[:, :k] + noise * torch.randn((b, k, v), generator=gen)).to(dtype)
    target = target.to(dtype)
    temp = 0.3 + torch.rand(b, generator=gen) if temps else None
    t = temp[:, None, None] if temps else 1.0
    ids = torch.zeros((b, k), dtype=torch.int64)
    if k:
        p = torch.softmax(dl.double() / t, -1)
        ids = torch.multinomial(p.reshape(b * k, v), 1, generator=gen).reshape(b, k)
    for s in greedy:
        temp[s] = 0.0
        best = target[s, :k].float().argmax(-1)
        ids[s] = torch.where(torch.rand(k, generator=gen) < 0.7, best, ids[s])
    nd = torch.randint(0, k + 3, (b,), generator=gen) if ragged else None
    return dict(target=target, ids=ids, au=torch.rand((b, k), generator=gen),
                su=torch.rand(b, generator=gen), draft=dl if draft else None, nd=nd, temp=temp)


def call(device, p, **over):
    a = {**p, **over}
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    u = lambda t: None if t is None else t.to(torch.int32).view(torch.uint32).to(device)  # noqa: E731
    return vpa.verify_draft_tokens(to(a["target"]), u(a["ids"]), to(a["au"]), to(a["su"]),
                                   draft_logits=to(a["draft"]), num_drafts=u(a["nd"]),
                                   temperature=to(a["temp"]))


def want(p):
    n = lambda t: None if t is None else (t.double().numpy() if t.is_floating_point()  # noqa: E731
                                          else t.numpy())
    return ref.verify(n(p["target"]), n(p["ids"]), n(p["au"]), n(p["su"]), n(p["draft"]), n(p["nd"]),
                      n(p["temp"]))


def check(device, p):
    ids, count, margin = want(p)
    assert np.all(margin > MARGIN), "a decision of this fixed input lies on its border"
    got, n = call(device, p)
    assert np.array_equal(n.cpu().numpy(), count)
    assert np.array_equal(got.cpu().numpy(), ids)
    return count


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 7, 64, 4095, 4096, 4097, 12345])
@pytest.mark.parametrize("k", [0, 1, 4])
@pytest.mark.parametrize("draft", [True, False])
def test_shapes(device, dtype, v, k, draft):
    p = problem(dtype, 9, k, v, draft=draft, seed=v + k, ragged=True)
    check(device, p)


@pytest.mark.parametrize("draft", [True, False])
def test_large_vocabulary(device, draft):
    p = problem(torch.bfloat16, 6, 4, 151936, draft=draft, seed=3, greedy=(2,))
    check(device, p)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,k,v", [(600, 3, 50), (300, 3, 4097), (700, 1, 8200)])
def test_many_sequences(device, dtype, b, k, v):
    """4096 segments and more: a wave each, with odd logits among them."""
    p = problem(dtype, b, k, v, draft=True, seed=b, ragged=True, greedy=(2, 5, b - 1))
    p["target"][9, 0, ::2] = float("nan")
    p["target"][10, 0] = torch.finfo(dtype).min
    p["target"][11, 0, 7] = float("inf")
    p["target"][12, 0] = float("-inf")
    check(device, p)


def test_flat_rows_of_a_large_vocabulary(device):
    """Every token about as likely as the next: the draw's sum has 100 000 borders."""
    p = problem(torch.float32, 24, 1, 100003, draft=True, spread=0.01, noise=0.01, seed=4)
    check(device, p)
    p = problem(torch.float32, 24, 0, 100003, spread=0.01, seed=5)
    check(device, p)


def test_most_drafts(device):
    """64 drafts, all accepted, none and some."""
    p = problem(torch.float32, 3, 64, 50, noise=0.0, seed=6)
    p["au"][0] = 0.0
    p["au"][1, 0] = 0.999999
    p["draft"][1, 0] = -5.0
    p["draft"][1, 0, int(p["ids"][1, 0])] = 30.0
    p["au"][2] *= 0.9
    count = check(device, p)
    assert count[0] == 65 and count[1] == 1


def test_equal_distributions_accept_and_fall_back(device):
    """p = q: accepted for every u < 1; a forced rejection draws from p."""
    p = problem(torch.float32, 4, 2, 300, noise=0.0, seed=7)
    ids, count = call(device, p)
    assert (count.cpu().numpy() == 3).all()
    got, n = call(device, p, au=torch.full((4, 2), 1.5))  # (beyond the range on purpose)
    for s in range(4):
        assert int(n.cpu()[s]) == 1
        r = ref.softmax(p["target"][s, 0].double().numpy(), float(p["temp"][s]))
        assert int(got.cpu()[s, 0]) == ref.draw(r, float(p["su"][s]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_and_odd_logits(device, dtype):
    p = problem(dtype, 12, 2, 5000, draft=True, seed=8)
    t, d = p["target"], p["draft"]
    inf, nan = float("inf"), float("nan")
    gen = torch.Generator().manual_seed(1)
    for s in range(12):
        hide = torch.rand((3, 5000), generator=gen) < 0.7
        t[s][hide] = -inf if s % 2 else nan
        d[s][torch.rand((2, 5000), generator=gen) < 0.5] = -inf
    t[4, 0] = -inf                      # nothing left: id 0
    t[5, 0] = nan
    t[6, 0, 17] = inf                   # takes all
    p["ids"][6, 0] = 17
    t[7, 0] = torch.finfo(dtype).min    # a mask of the type's lowest value everywhere: flat
    d[8, 0] = -inf                      # the drafter had nothing
    p["ids"][9, 0] = 5000               # ids past the vocabulary
    p["ids"][10, 1] = 2 ** 31 - 1
    ids, count, margin = want(p)
    got, n = call(device, p)
    for s in range(12):
        assert margin[s] > MARGIN
        assert np.array_equal(got.cpu().numpy()[s], ids[s]), s
    assert int(got.cpu()[4, 0]) == 0 and int(got.cpu()[5, 0]) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_greedy(device, dtype):
    """Temperatures of 0, below and NaN; ties go to the first; the answer is the argmax
    op's."""
    b, k, v = 9, 3, 9000
    p = problem(dtype, b, k, v, seed=9, draft=False, greedy=range(b))
    p["target"] = (2 * p["target"]).round() / 2  # many ties
    best = p["target"].float().argmax(-1)
    p["ids"] = torch.where(torch.rand((b, k), generator=torch.Generator().manual_seed(2)) < 0.7,
                           best[:, :k], p["ids"])
    p["temp"][3], p["temp"][4] = -1.0, float("nan")
    p["target"][5, 0, :9] = float("nan")
    count = check(device, p)
    assert len(set(count.tolist())) > 1
    rows = p["target"].reshape(-1, v).to(device)
    arg = vpa.argmax_token_ids_from_logits(rows).cpu().numpy().reshape(b, k + 1)
    got, n = call(device, p)
    for s in (0, 1, 2, 6, 7, 8):
        c = int(n.cpu()[s])
        assert int(got.cpu()[s, c - 1]) == arg[s, c - 1]


def test_extreme_temperatures(device):
    p = problem(torch.float32, 4, 1, 700, seed=10)
    p["temp"] = torch.tensor([1e-39, 1e30, float("inf"), 1e-3])
    for s in range(4):
        p["ids"][s, 0] = int(p["target"][s, 0].argmax())
    got, n = call(device, p)
    ids, count, margin = want(p)
    for s in range(4):
        if margin[s] > MARGIN:
            assert np.array_equal(got.cpu().numpy()[s], ids[s]), s


def test_unaligned_and_strided_rows(device):
    p = problem(torch.bfloat16, 5, 2, 4099, seed=11, ragged=True)
    a, n = call(device, p)
    for pad, shift in ((13, 3), (5, 0), (8, 8)):
        big = torch.zeros((5, 4, 4099 + pad + 11), dtype=torch.bfloat16, device=device)
        tv = big[:, :3, shift:shift + 4099]
        tv.copy_(p["target"])
        dbig = torch.zeros((5, 2, 4099 + pad + 7), dtype=torch.bfloat16, device=device)
        dv = dbig[..., shift:shift + 4099]
        dv.copy_(p["draft"])
        got, m = call(device, p, target=tv, draft=dv)
        assert torch.equal(got, a) and torch.equal(m, n)
    ids, count, _ = want(p)
    assert np.array_equal(a.cpu().numpy(), ids)


def test_one_row_for_all_sequences(device):
    """Rows repeated through zero strides."""
    p = problem(torch.float32, 1, 0, 900, seed=12, temps=False)
    su = torch.rand(50, generator=torch.Generator().manual_seed(3))
    rows = p["target"].to(device).expand(50, 1, 900)
    got, _ = vpa.verify_draft_tokens(rows, torch.zeros((50, 0), dtype=torch.uint32, device=device),
                                     torch.zeros((50, 0), device=device), su.to(device))
    r = ref.softmax(p["target"][0, 0].double().numpy(), 1.0)
    assert got.cpu().numpy()[:, 0].tolist() == [ref.draw(r, float(u)) for u in su]


def test_emitted_tokens_follow_the_target(device):
    """Over 40 000 sequences of one draft each, the first emitted token is distributed as
    the target's, whatever drafted it: chi-square over 8 tokens, 7 degrees of freedom, below
    24.3 (0.001; fixed seed)."""
    b, v = 40000, 8
    gen = torch.Generator().manual_seed(5)
    target = torch.randn((1, 1, v), generator=gen)
    dl = torch.randn((1, 1, v), generator=gen)
    q = torch.softmax(dl[0, 0].double(), -1)
    ids = torch.multinomial(q, b, replacement=True, generator=gen)[:, None]
    p = dict(target=target.expand(b, 2, v), ids=ids, au=torch.rand((b, 1), generator=gen),
             su=torch.rand(b, generator=gen), draft=dl.expand(b, 1, v), nd=None, temp=None)
    got, n = call(device, p)
    first = got.cpu().numpy()[:, 0]
    exp = torch.softmax(target[0, 0].double(), -1).numpy() * b
    chi = ((np.bincount(first, minlength=v) - exp) ** 2 / exp).sum()
    assert chi < 24.3
    assert 0.3 < (n.cpu().numpy() == 2).mean() < 1.0


def test_graph_replays(device):
    p = problem(torch.bfloat16, 7, 3, 6001, seed=13)
    dev = {k: (v.to(device) if v is not None and v.is_floating_point() else v) for k, v in p.items()}
    ids = p["ids"].to(torch.int32).view(torch.uint32).to(device)
    out = (torch.empty((7, 4), dtype=torch.uint32, device=device),
           torch.empty(7, dtype=torch.uint32, device=device))
    ws = vpa.verify_draft_tokens_workspace(7, 3, 6001, device)

    def step(out, ws):
        vpa.verify_draft_tokens(dev["target"], ids, dev["au"], dev["su"], draft_logits=dev["draft"],
                                temperature=dev["temp"], out=out, workspace=ws)

    step(out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out, ws)
    mine = (torch.empty_like(out[0]), torch.empty_like(out[1]))
    for i in range(4):
        dev["au"].uniform_()
        dev["su"].uniform_()
        dev["target"].mul_(0.97)
        step(mine, torch.empty_like(ws))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], mine[0]) and torch.equal(out[1], mine[1])
