"""What a decode loop does around the paged cache, as measurable cases.

* ``rotary_qk``      positions of several axes applied to new q and k rows (slices of one
                     projection), with the rows' RMS norms where the model has them.
* ``rotary_append``  the same, k and v written straight into the paged cache.
* ``weights``        the attention weight each cached token got, added to running scores.
* ``evict``          the cache cut to a budget of tokens by those scores.
* ``verify``         drafted tokens accepted or replaced from the target's logits.

``run`` computes them with elementary torch operations where ``own`` is false, and through
this package's entry points where it is true; ``exact`` restates them in 64 bits.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

_PKG = os.path.abspath("qwen3asr.rs_amd")
_TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_K_SCALE, _V_SCALE = 4.5 / 448.0, 4.0 / 448.0  # values to about 4.5 standard deviations
_EPS = 1e-6
_NONE = 0xFFFFFFFF  # an id or index past the last one


def _vpa():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import vpa

    return vpa


# ---- cases ----------------------------------------------------------------------------


def _case(name, kind, **over):
    c = {"name": name, "kind": kind, "dtype": "bf16"}
    if kind in ("rotary_qk", "rotary_append"):
        # one batch of new rows: `tokens` rows of the packed projection, positions below `far`
        c.update(tokens=1, heads=16, kv_heads=8, head_dim=128, rotary_dim=128, sections="24,20,20",
                 interleaved=True, adjacent=False, norm=True, theta=1e6, far=32768)
    if kind == "rotary_append":
        # `run_len` consecutive tokens of a sequence each (1: a decode step)
        c.update(block_size=16, fp8=False, run_len=1)
    if kind == "weights":
        c.update(heads=16, kv_heads=8, head_dim=128, block_size=16, fp8=False, batch=1,
                 rule="uniform", lo=512, hi=512, rows=1, lens_seed=1)
    if kind == "evict":
        c.update(kv_heads=8, head_dim=128, block_size=16, fp8=False, batch=1, lo=512, hi=512,
                 budget=256, first=4, last=64, lens_seed=1)
    if kind == "verify":
        # `batch` sequences with up to `drafts` drafted tokens each
        c.update(batch=1, drafts=4, vocab=151936, draft_logits=True, greedy=False, ragged=False)
    c.update(over)
    return c


def listed():
    return [
        # the smallest call: one token of one request, rotated in its own launch
        _case("rotary_qk_one", "rotary_qk"),
        # a prompt of a recording, far positions, rows without norms, half of the head rotated
        _case("rotary_qk_prompt", "rotary_qk", tokens=4500, dtype="f16", rotary_dim=64,
              sections="12,10,10", interleaved=False, norm=False, far=1000000),
        # a loaded server's decode step: one new token of 256 requests, each in a block of its own
        _case("rotary_append_decode256", "rotary_append", tokens=256),
        # admission of a batch: 64 requests of 512 new tokens
        _case("rotary_append_prefill", "rotary_append", tokens=32768, run_len=512),
        # one stream that sums the weights of every step
        _case("weights_one", "weights", lo=1500, hi=1500),
        # the loaded server's batch with its geometric length mix, one new token each
        _case("weights_decode256", "weights", batch=256, rule="geom", lo=800, hi=4096, lens_seed=5),
        # the last 32 rows of long prompts, as a cache is cut right after its prefill
        _case("weights_window", "weights", batch=8, lo=1000, hi=6000, rows=32, dtype="f16",
              lens_seed=3),
        # one long recording cut to half
        _case("evict_one_long", "evict", lo=8192, hi=8192, budget=4096, last=256),
        # a batch of mixed lengths cut to 1024 tokens, some of them shorter
        _case("evict_batch64", "evict", batch=64, lo=600, hi=4096, budget=1024, lens_seed=4),
        # one stream whose drafts were looked up in the text (no distribution of their own)
        _case("verify_one", "verify", draft_logits=False),
        # 64 streams, four drafts each with the drafting model's logits
        _case("verify_batch64", "verify", batch=64),
        # greedy verification of a large batch, drafts of uneven length
        _case("verify_greedy128", "verify", batch=128, drafts=3, greedy=True, draft_logits=False,
              ragged=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary_qk", "rotary_append", "weights", "evict", "verify"])
    c = _case("", kind)
    del c["name"]
    c["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("rotary_qk", "rotary_append"):
        c["heads"], c["kv_heads"] = rng.choice([(16, 8), (16, 8), (32, 8), (24, 8), (16, 16), (14, 2)])
        c["head_dim"] = rng.choice([64, 96, 128, 128, 192, 256])
        c["rotary_dim"] = rng.choice([c["head_dim"], c["head_dim"], c["head_dim"] // 2])
        half = c["rotary_dim"] // 2
        h = half * 5 // 16
        c["sections"] = rng.choice(["%d" % half, "%d,%d,%d" % (half - 2 * h, h, h)])
        c["interleaved"] = rng.random() < 0.5
        c["adjacent"] = rng.random() < 0.25
        c["norm"] = rng.random() < 0.6
        c["theta"] = rng.choice([1e4, 1e6, 5e6])
        c["far"] = _log_int(rng, 512, 1000000)
        room = 32768 * 32 * 256 // ((c["heads"] + 2 * c["kv_heads"]) * c["head_dim"] * _BYTES[c["dtype"]])
        c["tokens"] = _log_int(rng, 1, min(room, 32768))
    if kind == "rotary_append":
        c["block_size"] = rng.choice([8, 16, 16, 32])
        c["fp8"] = rng.random() < 0.3
        c["run_len"] = rng.choice([1, _log_int(rng, 2, 1024)])
        if c["run_len"] == 1:
            c["tokens"] = min(c["tokens"], 1024)
    if kind in ("weights", "evict"):
        c["block_size"] = rng.choice([8, 16, 16, 32])
        c["head_dim"] = rng.choice([64, 96, 128, 128, 192, 256])
        c["lens_seed"] = rng.randrange(1, 1 << 20)
        c["fp8"] = rng.random() < 0.25
        c["batch"] = _log_int(rng, 1, 256 if kind == "weights" else 64)
        room = (160000 if kind == "weights" else 120000) * 128 * 2 // (
            c["batch"] * c["head_dim"] * _BYTES[c["dtype"]])
        c["hi"] = _log_int(rng, 64, max(64, min(8192, room)))
        c["lo"] = rng.randrange(1, c["hi"] + 1)
    if kind == "weights":
        c["heads"], c["kv_heads"] = rng.choice([(16, 8), (16, 8), (32, 8), (24, 8), (8, 8), (14, 2)])
        c["rows"] = rng.choice([1, 1, rng.randrange(2, 9), rng.randrange(9, 33)])
        if c["rows"] > 8:
            c["batch"] = min(c["batch"], 8)
    if kind == "evict":
        c["budget"] = _log_int(rng, 16, max(16, c["hi"]))
        c["first"] = rng.randrange(0, 1 + min(8, c["budget"] // 4))
        c["last"] = rng.randrange(0, 1 + c["budget"] // 2)
    if kind == "verify":
        c["batch"] = _log_int(rng, 1, 64)
        c["drafts"] = rng.randrange(0, 9)
        c["vocab"] = rng.choice([151936, 151936, _log_int(rng, 500, 150000)])
        c["greedy"] = rng.random() < 0.25
        c["draft_logits"] = not c["greedy"] and rng.random() < 0.6
        c["ragged"] = rng.random() < 0.5
        while work(c)["bytes"] > 180e6:
            c["batch"] = max(1, c["batch"] // 2)
    return c


# ---- sizes, from the case alone ---------------------------------------------------------


def _lens(case):
    rng = np.random.default_rng(case["lens_seed"])
    if case.get("rule") == "geom":
        n = np.clip(rng.geometric(1.0 / case["lo"], size=case["batch"]), 16, case["hi"])
    else:
        n = rng.integers(case["lo"], case["hi"], size=case["batch"], endpoint=True)
    return np.maximum(n, 1).astype(np.int64)


def _rows(case, lens):
    """Query rows of each sequence: at most its tokens."""
    return np.minimum(lens, case["rows"])


def work(case):
    e = _BYTES[case["dtype"]]
    if case["kind"] in ("rotary_qk", "rotary_append"):
        t, d, r = case["tokens"], case["head_dim"], case["rotary_dim"]
        hq, hk = case["heads"], case["kv_heads"]
        axes = len(case["sections"].split(","))
        flops = t * (hq + hk) * (3 * r + (4 * d if case["norm"] else 0))
        if case["kind"] == "rotary_qk":
            return {"bytes": 2 * t * (hq + hk) * d * e + 8 * axes * t, "flops": flops}
        c = 1 if case["fp8"] else e
        return {"bytes": t * d * (2 * hq * e + 2 * hk * (e + c)) + 8 * (axes + 1) * t, "flops": flops}
    if case["kind"] == "verify":
        b, k, v = case["batch"], case["drafts"], case["vocab"]
        rows = b * (k + 1) + (b * k if case["draft_logits"] else 0)
        return {"bytes": rows * v * e + 4 * b * (3 * k + 3), "flops": (1 if case["greedy"] else 4) * rows * v}
    lens = _lens(case)
    c = 1 if case["fp8"] else e
    row = case["kv_heads"] * case["head_dim"]
    if case["kind"] == "weights":
        n = _rows(case, lens)
        q = case["heads"] * case["head_dim"]
        return {"bytes": int(lens.sum()) * (row * c + 8 * case["kv_heads"]) + int(n.sum()) * q * e
                + 4 * int((-(-lens // case["block_size"])).sum()),
                "flops": 2 * q * int((n * lens).sum()) + 4 * case["heads"] * int((n * lens).sum())}
    cut = lens > case["budget"]
    moved = int(cut.sum()) * (case["budget"] - case["first"])
    return {"bytes": 4 * moved * row * c + 4 * case["kv_heads"] * int((2 * lens * cut).sum())
            + 4 * case["kv_heads"] * int(np.minimum(lens, case["budget"]).sum()),
            "flops": case["kv_heads"] * int(lens.sum())}


# ---- inputs -----------------------------------------------------------------------------


def _axes(case):
    """Axis of each rotated pair, [rotary_dim / 2]."""
    half = case["rotary_dim"] // 2
    sec = [int(n) for n in case["sections"].split(",")]
    a = np.zeros(half, np.uint8)
    if case["interleaved"]:  # t h w t h w ..., the rest t
        for k in range(1, len(sec)):
            a[k:len(sec) * sec[k]:len(sec)] = k
        return a
    return np.repeat(np.arange(len(sec)), sec).astype(np.uint8)


def _caches(case, nb, rand):
    d, bs, kvh = case["head_dim"], case["block_size"], case["kv_heads"]
    x = 16 if case["fp8"] else 16 // _BYTES[case["dtype"]]
    kc, vc = rand(nb, kvh, d // x, bs, x), rand(nb, kvh, d, bs)
    if not case["fp8"]:
        return kc, vc, None, None
    ks = torch.tensor([_K_SCALE], dtype=torch.float32, device=kc.device)
    vs = torch.tensor([_V_SCALE], dtype=torch.float32, device=kc.device)
    return ((kc.float() / ks).clamp_(-448, 448).to(torch.float8_e4m3fn),
            (vc.float() / vs).clamp_(-448, 448).to(torch.float8_e4m3fn), ks, vs)


def _tables(rng, lens, bs):
    """Block tables of sequences of these lengths over shuffled blocks 1.., and the pool's size."""
    need = -(-lens // bs)
    nb = int(need.sum()) + 1 + int(need.sum()) // 8
    ids = rng.permutation(np.arange(1, nb))
    t = np.zeros((len(lens), int(need.max())), np.uint32)
    at = np.concatenate([[0], np.cumsum(need)])
    for s in range(len(lens)):
        t[s, :need[s]] = ids[at[s]:at[s + 1]]
    return t, nb


def prepare(case, seed):
    dev = torch.device("cuda")
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dt = _TORCH[case["dtype"]]

    def rand(*shape):
        return torch.empty(shape, dtype=dt, device=dev).normal_(generator=gen)

    s = {"case": case}
    if case["kind"] in ("rotary_qk", "rotary_append"):
        t, h, kvh, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
        qkv = rand(t, (h + 2 * kvh) * d)  # one projection's output
        s["q"] = qkv[:, :h * d].view(t, h, d)
        s["k"] = qkv[:, h * d:(h + kvh) * d].view(t, kvh, d)
        s["v"] = qkv[:, (h + kvh) * d:].view(t, kvh, d)
        axes = _axes(case)
        s["axes"] = torch.from_numpy(axes).to(dev)
        s["inv_freq"] = torch.from_numpy(
            case["theta"] ** -(np.arange(0, case["rotary_dim"], 2) / case["rotary_dim"])).to(dev)
        s["positions"] = torch.from_numpy(
            rng.integers(0, case["far"], size=(int(axes.max()) + 1, t))).to(dev)
        s["qw"] = s["kw"] = None
        if case["norm"]:
            s["qw"] = (1 + 0.2 * rand(d).float()).to(dt)
            s["kw"] = (1 + 0.2 * rand(d).float()).to(dt)
    if case["kind"] == "rotary_append":
        bs, n = case["block_size"], case["run_len"]
        runs = -(-t // n)
        prior = np.random.default_rng(t).integers(0, 4 * bs, size=runs)  # the pool's size: the case's
        lens = prior + np.minimum(n, t - n * np.arange(runs))
        tables, nb = _tables(rng, lens, bs)
        which = np.arange(t) // n
        pos = prior[which] + np.arange(t) % n
        s["slots"] = torch.from_numpy(tables[which, pos // bs].astype(np.int64) * bs + pos % bs).to(dev)
        s["kc"], s["vc"], s["ks"], s["vs"] = _caches(case, nb, rand)
    if case["kind"] in ("weights", "evict"):
        lens = _lens(case)
        tables, nb = _tables(rng, lens, case["block_size"])
        s["kc"], s["vc"], s["ks"], s["vs"] = _caches(case, nb, rand)
        s["tables"] = torch.from_numpy(tables).to(dev)
        s["lens"] = torch.from_numpy(lens.astype(np.uint32)).to(dev)
        s["max_len"] = int(lens.max())
        wide = tables.shape[1] * case["block_size"]
        # weights so far: heavy-tailed, as sums of softmax rows are
        s["scores"] = torch.empty((len(lens), case["kv_heads"], wide), device=dev).normal_(
            generator=gen).mul_(1.5).exp_().mul_(0.01)
    if case["kind"] == "weights":
        del s["vc"]
        n = _rows(case, lens)
        s["max_rows"] = int(n.max())
        s["cu"] = torch.from_numpy(np.concatenate([[0], np.cumsum(n)]).astype(np.uint32)).to(dev)
        s["q"] = rand(int(n.sum()), case["heads"], case["head_dim"])
    if case["kind"] == "verify":
        b, k, v = case["batch"], case["drafts"], case["vocab"]
        # peaked rows over a long tail; the drafting model agrees with the target up to noise
        target = torch.empty((b, k + 1, v), device=dev).normal_(generator=gen).mul_(2.5)
        draft = target[:, :k] + 0.7 * torch.empty((b, k, v), device=dev).normal_(generator=gen)
        s["target"] = target.to(dt)
        s["draft"] = draft.to(dt) if case["draft_logits"] else None
        s["temperature"] = torch.zeros(b, device=dev) if case["greedy"] else torch.empty(
            b, device=dev).uniform_(0.3, 1.1, generator=gen)
        if case["greedy"]:  # mostly the target's own choice
            ids = s["target"][:, :k].float().argmax(-1)
            other = torch.randint(0, v, (b, k), generator=gen, device=dev)
            ids = torch.where(torch.rand((b, k), generator=gen, device=dev) < 0.7, ids, other)
        else:
            p = torch.softmax((draft.to(dt).float() / s["temperature"][:, None, None]), -1)
            ids = torch.multinomial(p.reshape(b * k, v), 1, generator=gen).reshape(b, k) if k else \
                torch.zeros((b, 0), dtype=torch.int64, device=dev)
        s["draft_ids"] = ids.to(torch.int32).view(torch.uint32)
        s["accept_u"] = torch.rand((b, k), generator=gen, device=dev)
        s["sample_u"] = torch.rand(b, generator=gen, device=dev)
        s["num_drafts"] = None
        if case["ragged"]:
            s["num_drafts"] = torch.from_numpy(rng.integers(0, k + 1, size=b).astype(np.uint32)).to(dev)
    return s


# ---- one pass ---------------------------------------------------------------------------


def run(s):
    kind = s["case"]["kind"]
    if own:
        return _run_own(_vpa(), s, kind)
    return _PLAIN[kind](s)


def _run_own(vpa, s, kind):
    case = s["case"]
    if kind == "rotary_qk":
        q, k = vpa.rotary_qk(s["q"], s["k"], s["positions"], s["inv_freq"], s["axes"],
                             q_norm=s["qw"], k_norm=s["kw"], norm_eps=_EPS,
                             adjacent=case["adjacent"])
        return {"q": q, "k": k}
    if kind == "rotary_append":
        q = vpa.rotary_reshape_and_cache(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"],
                                         s["axes"], s["ks"], s["vs"], s["kc"], s["vc"], s["slots"],
                                         q_norm=s["qw"], k_norm=s["kw"], norm_eps=_EPS,
                                         adjacent=case["adjacent"])
        return {"q": q, "key_cache": s["kc"], "value_cache": s["vc"]}
    if kind == "weights":
        vpa.paged_attention_weights(s["q"], s["kc"], s["ks"], s["tables"], s["lens"],
                                    case["head_dim"] ** -0.5, s["scores"], cu_seqlens_q=s["cu"],
                                    max_query_len=s["max_rows"], max_context_len=s["max_len"])
        return s["scores"]
    if kind == "evict":
        lens, kept = vpa.evict_kv_cache(s["kc"], s["vc"], s["scores"], s["tables"], s["lens"],
                                        case["budget"], keep_first=case["first"],
                                        keep_last=case["last"], max_context_len=s["max_len"])
        return {"lens": lens.view(torch.int32), "kept": kept.view(torch.int32),
                "scores": s["scores"], "key_cache": s["kc"], "value_cache": s["vc"]}
    ids, count = vpa.verify_draft_tokens(s["target"], s["draft_ids"], s["accept_u"], s["sample_u"],
                                         draft_logits=s["draft"], num_drafts=s["num_drafts"],
                                         temperature=s["temperature"])
    return {"ids": ids.view(torch.int32), "count": count.view(torch.int32)}


def _plain_rotate(s):
    """q and k normalised and rotated, in 32 bits; the angles in 64."""
    case = s["case"]
    half = case["rotary_dim"] // 2
    pos = s["positions"][s["axes"].long()]  # [half, T]
    angle = (pos.double() * s["inv_freq"][:, None]).t()[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def turn(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w.float()
        if case["adjacent"]:
            a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
            y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = x[..., :half], x[..., half:2 * half]
            y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((y, x[..., 2 * half:]), -1)

    return turn(s["q"], s["qw"]), turn(s["k"], s["kw"])


def _plain_rotary_qk(s):
    q, k = _plain_rotate(s)
    return {"q": q.to(s["q"].dtype), "k": k.to(s["k"].dtype)}


def _plain_rotary_append(s):
    case = s["case"]
    q, k = _plain_rotate(s)
    v = s["v"]
    if case["fp8"]:
        k, v = (k / s["ks"]).clamp(-448, 448), (v.float() / s["vs"]).clamp(-448, 448)
    k, v = k.to(s["kc"].dtype), v.to(s["vc"].dtype)
    bs = case["block_size"]
    blk, off = s["slots"] // bs, s["slots"] % bs
    t, kvh, d = k.shape
    x = s["kc"].shape[-1]
    kc, vc = s["kc"], s["vc"]
    k = k.reshape(t, kvh, d // x, x)
    if case["fp8"]:  # bytes are indexed as bytes
        kc, vc, k, v = (a.view(torch.uint8) for a in (kc, vc, k, v))
    kc[blk, :, :, off] = k
    vc[blk, :, :, off] = v
    return {"q": q.to(s["q"].dtype), "key_cache": s["kc"], "value_cache": s["vc"]}


def _plain_weights(s):
    case = s["case"]
    kvh, d, n_max, l_max = case["kv_heads"], case["head_dim"], s["max_rows"], s["max_len"]
    group = case["heads"] // kvh
    dev = s["q"].device
    lens, cu = s["lens"].view(torch.int32).long(), s["cu"].view(torch.int32).long()
    b = lens.shape[0]
    cols = -(-l_max // case["block_size"])
    k = s["kc"][s["tables"].view(torch.int32).long()[:, :cols]].float()  # [b, cols, kvh, d/x, bs, x]
    if case["fp8"]:
        k = k * s["ks"]
    k = k.permute(0, 2, 3, 5, 1, 4).reshape(b, kvh, d, -1)[..., :l_max].contiguous()
    row = torch.arange(n_max, device=dev)
    n = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + row).clamp_(max=s["q"].shape[0] - 1)
    q = s["q"][at].float().reshape(b, n_max, kvh, group, d).permute(0, 2, 3, 1, 4)
    logits = torch.matmul(q.reshape(b, kvh, group * n_max, d), k) * d ** -0.5
    logits = logits.reshape(b, kvh, group, n_max, l_max)
    tok = torch.arange(l_max, device=dev)
    seen = (tok[None, None] <= (row[None] + (lens - n)[:, None])[..., None]) & (row[None] < n[:, None])[..., None]
    logits = logits.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = torch.where(seen[:, None, None], p / p.sum(-1, keepdim=True), 0.0)
    s["scores"][..., :l_max] += p.sum((2, 3))
    return s["scores"]


def _plain_evict(s):
    case = s["case"]
    dev, bs, most = s["kc"].device, case["block_size"], case["budget"]
    lens = s["lens"].view(torch.int32).long()
    b, kvh, wide = s["scores"].shape
    tok = torch.arange(wide, device=dev)
    inside = tok < lens[:, None]
    forced = (tok < case["first"]) | (tok >= (lens - case["last"])[:, None])
    score = s["scores"]
    # rank: kept in any case, then numbers from the highest down, then NaN; ties by place
    tier = torch.where(forced[:, None], 0, torch.where(torch.isnan(score), 2, 1))
    tier = torch.where(inside[:, None], tier, 3)
    order = torch.sort(torch.nan_to_num(score, nan=0.0, posinf=math.inf, neginf=-math.inf), dim=-1,
                       descending=True, stable=True).indices
    order = order.gather(-1, torch.sort(tier.gather(-1, order), dim=-1, stable=True).indices)
    new = lens.clamp(max=most)
    rank = torch.arange(most, device=dev)
    order = order[..., :most]
    if order.shape[-1] < most:
        order = torch.cat((order, order.new_zeros(b, kvh, most - order.shape[-1])), -1)
    valid = (rank < new[:, None])[:, None].expand(b, kvh, most)
    kept = torch.where(valid, order, wide + 1).sort(-1).values
    src = torch.where(valid, kept, rank).clamp_(max=wide - 1)
    dst = rank.clamp(max=wide - 1).expand(b, kvh, most)
    tables = s["tables"].view(torch.int32).long()
    head = torch.arange(kvh, device=dev)[None, :, None].expand(b, kvh, most)

    def block(t):
        return tables.gather(1, (t // bs).reshape(b, -1)).reshape(b, kvh, most)

    at, to = (block(src), head, slice(None), src % bs), (block(dst), head, slice(None), dst % bs)
    kc, vc = s["kc"], s["vc"]
    if case["fp8"]:  # bytes are indexed as bytes
        kc, vc = kc.view(torch.uint8), vc.view(torch.uint8)
    kc[to] = kc[at]
    vc[to] = vc[at]
    short = torch.where(valid, score.gather(-1, src), 0.0)[..., :wide]
    moved = torch.nn.functional.pad(short, (0, max(0, wide - short.shape[-1])))
    score.copy_(torch.where(inside[:, None], moved, score))
    return {"lens": new.to(torch.int32), "kept": torch.where(valid, kept, -1).to(torch.int32),
            "scores": score, "key_cache": s["kc"], "value_cache": s["vc"]}


def _plain_verify(s):
    # probabilities in 64 bits: the results are whole numbers next to borders of sums
    case = s["case"]
    b, k, v = case["batch"], case["drafts"], case["vocab"]
    dev = s["target"].device
    n = s["num_drafts"].view(torch.int32).long() if s["num_drafts"] is not None else \
        torch.full((b,), k, device=dev)
    ids = s["draft_ids"].view(torch.int32).long()
    step = torch.arange(k, device=dev)
    if case["greedy"]:
        best = s["target"].float().argmax(-1)  # [b, k + 1]
        good = best[:, :k] == ids
    else:
        t = s["temperature"].double()[:, None, None]
        p = torch.softmax(s["target"].double() / t, -1)
        px = p[:, :k].gather(-1, ids[..., None])[..., 0]
        qx = 1.0
        if s["draft"] is not None:
            q = torch.softmax(s["draft"].double() / t, -1)
            qx = q.gather(-1, ids[..., None])[..., 0]
        good = s["accept_u"].double() * qx < px
    good = good & (step < n[:, None])
    took = good.long().cumprod(-1).sum(-1)  # accepted drafts
    if case["greedy"]:
        last = best.gather(-1, took[:, None])[:, 0]
    else:
        row = torch.arange(b, device=dev)
        r = p[row, took]
        if k:
            at = took.clamp(max=k - 1)
            if s["draft"] is not None:
                left = (r - q[row, at]).clamp_(min=0)
                left = torch.where(left.sum(-1, keepdim=True) > 0, left, r)
            else:
                left = r.scatter(-1, ids[row, at][:, None], 0.0)
            r = torch.where((took < n)[:, None], left, r)
        upto = r.cumsum(-1)
        last = (upto > s["sample_u"].double()[:, None] * upto[:, -1:]).long().argmax(-1)
    place = torch.arange(k + 1, device=dev)
    out = torch.full((b, k + 1), -1, dtype=torch.int64, device=dev)
    if k:
        out[:, :k] = torch.where(step < took[:, None], ids, -1)
    out = torch.where(place == took[:, None], last[:, None], out)
    return {"ids": out.to(torch.int32), "count": (took + 1).to(torch.int32)}


_PLAIN = {"rotary_qk": _plain_rotary_qk, "rotary_append": _plain_rotary_append,
          "weights": _plain_weights, "evict": _plain_evict, "verify": _plain_verify}


# ---- the definitions in 64 bits -----------------------------------------------------------


def _exact_rotary(case, s):
    d, r = case["head_dim"], case["rotary_dim"]
    axis = _axes(case)
    first = np.arange(r // 2) * 2 if case["adjacent"] else np.arange(r // 2)
    second = first + 1 if case["adjacent"] else first + r // 2
    pos = s["positions"].cpu().numpy().astype(np.float64)
    freq = case["theta"] ** -(2.0 * np.arange(r // 2) / r)
    turn = np.zeros((case["tokens"], d), np.complex128)
    turn[:, first] = np.exp(1j * (pos[axis] * freq[:, None]).T)
    turn = torch.from_numpy(turn[:, first]).to("cuda")[:, None]

    def one(x, w):
        x = x.double()
        if w is not None:
            x = w.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / d + _EPS)
        z = torch.complex(x[..., first], x[..., second]) * turn
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    return one(s["q"], s["qw"]), one(s["k"], s["kw"])


def _exact_weights(case, s):
    lens, d = _lens(case), case["head_dim"]
    n = _rows(case, lens)
    kvh, bs = case["kv_heads"], case["block_size"]
    group = case["heads"] // kvh
    tables = s["tables"].view(torch.int32).long()
    out = s["scores"].double()
    a = 0
    for i in range(len(lens)):
        size, rows = int(lens[i]), int(n[i])
        k = s["kc"][tables[i, :-(-size // bs)]].double() * (float(s["ks"]) if case["fp8"] else 1.0)
        k = k.permute(1, 0, 3, 2, 4).reshape(kvh, -1, d)[:, :size]
        q = s["q"][a:a + rows].double().reshape(rows, kvh, group, d)
        a += rows
        for r in range(rows):
            see = size - rows + r + 1
            p = torch.softmax(torch.bmm(q[r], k[:, :see].transpose(1, 2).contiguous()) / math.sqrt(d), -1)
            out[i, :, :see] += p.sum(1)
    return out


def _exact_evict(case, s):
    lens, bs, kvh = _lens(case), case["block_size"], case["kv_heads"]
    score = s["scores"].cpu().numpy()
    tables = s["tables"].cpu().numpy().astype(np.int64)
    out, kc, vc = score.astype(np.float64), s["kc"].float(), s["vc"].float()
    k_new, v_new = kc.clone(), vc.clone()
    for i in range(len(lens)):
        size = int(lens[i])
        if size <= case["budget"]:
            continue
        low, high = min(case["first"], size), max(size - case["last"], case["first"])
        for j in range(kvh):
            middle = sorted(range(low, high), key=lambda t: (-score[i, j, t], t))
            keep = sorted(list(range(low)) + list(range(high, size)) +
                          middle[:case["budget"] - low - (size - high)])
            at, to = np.array(keep), np.arange(len(keep))
            src, dst = tables[i, at // bs], tables[i, to // bs]
            k_new[dst, j, :, to % bs] = kc[src, j, :, at % bs]
            v_new[dst, j, :, to % bs] = vc[src, j, :, at % bs]
            out[i, j, :size] = 0
            out[i, j, :len(keep)] = score[i, j, at]
    return {"lens": None, "kept": None, "scores": torch.from_numpy(out), "key_cache": k_new.double(),
            "value_cache": v_new.double()}


def exact(case, seed):
    if case["kind"] == "verify":
        return None  # whole numbers only
    s = prepare(case, seed)
    if case["kind"] == "weights":
        return _exact_weights(case, s)
    if case["kind"] == "evict":
        return _exact_evict(case, s)
    q, k = _exact_rotary(case, s)
    if case["kind"] == "rotary_qk":
        return {"q": q, "k": k}
    v = s["v"].double()
    if case["fp8"]:
        k, v = k / s["ks"].double(), v / s["vs"].double()
    kc, vc = s["kc"].double(), s["vc"].double()
    slot, bs = s["slots"].cpu().numpy(), case["block_size"]
    x = kc.shape[-1]
    kc[slot // bs, :, :, slot % bs] = k.reshape(k.shape[0], k.shape[1], -1, x)
    vc[slot // bs, :, :, slot % bs] = v
    return {"q": q, "key_cache": kc, "value_cache": vc}
