"""A serving loop with several continuations per request, as measurable cases.

* ``append``     new k and v rows into a cache of 8-bit values with a scale for each block of
                 tokens and head.
* ``attention``  attention over that cache: one new token, drafted tokens or a prompt's rows.
* ``fork``       rows of a batch continued as several, sharing the blocks that are full; the
                 copies are given up again.
* ``compact``    requests end, the blocks in use move to the front of the pool, others start.
* ``logits``     penalties for repeated tokens, biases and grammar masks, before a token is
                 chosen.

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
_TOP = 448.0  # largest finite E4M3 value
_LEAST = -100  # exponent of the smallest scale
_NONE = 0xFFFFFFFF  # no mask


def _vpa():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import vpa

    return vpa


# ---- cases ----------------------------------------------------------------------------


def _case(name, kind, **over):
    c = {"name": name, "kind": kind, "dtype": "bf16"}
    if kind in ("append", "attention"):
        c.update(kv_heads=8, head_dim=128, block_size=16)
    if kind == "append":
        # `run_len` consecutive tokens of a sequence each (1: a decode step)
        c.update(tokens=1, run_len=1)
    if kind == "attention":
        # up to `rows` query rows per sequence; scales that are powers of two, or any
        c.update(heads=16, batch=1, rule="uniform", lo=512, hi=512, rows=1, causal=True, pow2=True,
                 lens_seed=1)
    if kind in ("fork", "compact"):
        # caches of `layers` layers, in 8 bits with block scales or in 16 bits
        c.update(kv_heads=8, head_dim=128, block_size=16, layers=28, scaled=False, lens_seed=1)
    if kind == "fork":
        c.update(prompts=1, ways=4, lo=512, hi=512)
    if kind == "compact":
        # `rows` requests in a pool of `blocks`
        c.update(rows=8, blocks=512)
    if kind == "logits":
        # `batch` sequences, `drafts` drafted tokens each (0: one row per sequence)
        c.update(batch=1, drafts=0, vocab=151936, prompt=1500, generated=200, penalties=True,
                 biases=0, masks=0, allowed=0.5, lens_seed=1)
    c.update(over)
    return c


def listed():
    return [
        # a loaded server's decode step: one new token of 256 requests, each in a block of its own
        _case("append_decode256", "append", tokens=256),
        # admission of a batch: 64 requests of 512 new tokens
        _case("append_prefill", "append", tokens=32768, run_len=512),
        # one stream's decode step
        _case("attention_one", "attention", lo=1500, hi=1500),
        # the loaded server's batch with its geometric length mix
        _case("attention_decode256", "attention", batch=256, rule="geom", lo=800, hi=4096, lens_seed=5),
        # the next chunk of a long prompt, over what is cached
        _case("attention_chunk", "attention", lo=6512, hi=6512, rows=512, dtype="f16"),
        # 64 requests of 512 new tokens over shared or earlier ones
        _case("attention_prefill", "attention", batch=64, lo=560, hi=1600, rows=512, lens_seed=4),
        # one prompt sampled eight times
        _case("fork_samples", "fork", ways=8, lo=1500, hi=1500),
        # beams of 32 requests, three new ones each
        _case("fork_beams", "fork", prompts=32, ways=3, lo=300, hi=900, scaled=True, lens_seed=3),
        # a small pool after a few requests ended
        _case("compact_small", "compact", rows=8, blocks=256, scaled=True),
        # a larger one, to be cut to what is in use
        _case("compact_pool", "compact", rows=32, blocks=1024, lens_seed=2),
        # one stream with a repetition penalty
        _case("logits_one", "logits", dtype="f32", biases=8),
        # a batch with penalties, biases and a grammar for most rows
        _case("logits_batch256", "logits", batch=256, generated=512, biases=64, masks=16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "attention", "attention", "attention", "fork", "compact",
                       "logits", "logits"])
    c = _case("", kind)
    del c["name"]
    c["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
    c["lens_seed"] = rng.randrange(1, 1 << 20)
    if kind != "logits":
        c["block_size"] = rng.choice([8, 16, 16, 32])
        c["head_dim"] = rng.choice([64, 96, 128, 128, 192, 256])
        c["kv_heads"] = rng.choice([2, 4, 8, 8, 16])
    if kind == "append":
        room = 32768 * 8 * 128 * 3 // (c["kv_heads"] * c["head_dim"] * (_BYTES[c["dtype"]] + 1))
        c["tokens"] = _log_int(rng, 1, min(room, 32768))
        c["run_len"] = rng.choice([1, _log_int(rng, 2, 1024)])
        if c["run_len"] == 1:
            c["tokens"] = min(c["tokens"], 1024)
    if kind == "attention":
        c["heads"] = c["kv_heads"] * rng.choice([1, 2, 2, 3, 4, 7, 8])
        c["pow2"] = rng.random() < 0.5
        c["rows"] = rng.choice([1, 1, rng.randrange(2, 9), _log_int(rng, 9, 1024)])
        c["causal"] = rng.random() < 0.8
        c["batch"] = _log_int(rng, 1, 256 if c["rows"] <= 8 else 32)
        c["hi"] = _log_int(rng, 16, 8192)
        c["lo"] = rng.randrange(1, c["hi"] + 1)
        # as many keys, and products of rows with keys, as the largest listed ones
        while c["batch"] * c["hi"] * c["kv_heads"] * c["head_dim"] > 1.6e8 or \
                c["batch"] * min(c["rows"], c["hi"]) * c["hi"] * c["heads"] * c["head_dim"] > 6e10:
            if c["batch"] > 1:
                c["batch"] = (c["batch"] + 1) // 2
            else:
                c["hi"] = (c["hi"] + 1) // 2
                c["lo"] = min(c["lo"], c["hi"])
    if kind in ("fork", "compact"):
        c["scaled"] = rng.random() < 0.5
        c["layers"] = rng.randrange(1, 29)
        row = c["kv_heads"] * c["head_dim"] * c["block_size"] * 2 * (1 if c["scaled"] else 2)
        most = min(1024, int(1.6e9) // (row * c["layers"]))  # blocks
    if kind == "fork":
        c["prompts"] = _log_int(rng, 1, 32)
        c["ways"] = rng.randrange(1, 9)
        c["hi"] = _log_int(rng, 2, 2000)
        while c["prompts"] * (-(-c["hi"] // c["block_size"]) + c["ways"]) > most and c["hi"] > 1:
            if c["prompts"] > 1:
                c["prompts"] //= 2
            else:
                c["hi"] //= 2
        c["lo"] = rng.randrange(1, c["hi"] + 1)
    if kind == "compact":
        c["blocks"] = _log_int(rng, 16, max(16, most))
        c["rows"] = rng.randrange(2, 1 + max(2, min(64, c["blocks"] // 4)))
    if kind == "logits":
        c["batch"] = _log_int(rng, 1, 256)
        c["drafts"] = rng.choice([0, 0, rng.randrange(1, 5)])
        c["batch"] = max(1, c["batch"] // (c["drafts"] + 1))
        c["vocab"] = rng.choice([151936, 151936, _log_int(rng, 500, 150000)])
        c["prompt"] = rng.choice([0, _log_int(rng, 1, 6000)])
        c["generated"] = _log_int(rng, 1, 2000)
        c["penalties"] = rng.random() < 0.8
        c["biases"] = rng.choice([0, rng.randrange(1, 300)])
        c["masks"] = rng.choice([0, rng.randrange(1, 17)])
        c["allowed"] = rng.choice([0.001, 0.5, 0.99])
        if c["dtype"] == "f32":
            c["batch"] = max(1, c["batch"] // 2)
    return c


# ---- sizes, from the case alone ---------------------------------------------------------


def _lens(case, n):
    rng = np.random.default_rng(case["lens_seed"])
    if case.get("rule") == "geom":
        lens = np.clip(rng.geometric(1.0 / case["lo"], size=n), 16, case["hi"])
    else:
        lens = rng.integers(case["lo"], case["hi"], size=n, endpoint=True)
    return np.maximum(lens, 1).astype(np.int64)


def _rows(case, lens):
    """Query rows of each sequence: at most its tokens."""
    return np.minimum(lens, case["rows"])


def _runs(case):
    """Tokens that each appended-to sequence held before and holds afterwards."""
    runs = -(-case["tokens"] // case["run_len"])
    prior = np.random.default_rng(case["tokens"]).integers(0, 4 * case["block_size"], size=runs)
    return prior, prior + np.minimum(case["run_len"], case["tokens"] - case["run_len"] * np.arange(runs))


def _block_bytes(case):
    """Of one block over all layers and its buffers."""
    row = case["kv_heads"] * case["head_dim"] * case["block_size"]
    return 2 * case["layers"] * (row + 4 * case["kv_heads"] if case["scaled"] else 2 * row)


def _pool_rows(case):
    """Blocks of each request, in use and waiting, in a pool that a quarter of is free."""
    rng = np.random.default_rng(case["lens_seed"])
    share = rng.uniform(0.5, 1.5, size=case["rows"])
    n = np.floor(share / share.sum() * 0.75 * (case["blocks"] - 1)).astype(np.int64)
    return np.maximum(n, 1)


def work(case):
    e = _BYTES[case["dtype"]]
    if case["kind"] == "append":
        prior, lens = _runs(case)
        bs = case["block_size"]
        blocks = int((-(-lens // bs) - prior // bs).sum())
        n = 2 * case["tokens"] * case["kv_heads"] * case["head_dim"]
        return {"bytes": n * (e + 1) + 8 * case["tokens"] + 8 * case["kv_heads"] * blocks,
                "flops": 3 * n}
    if case["kind"] == "attention":
        lens = _lens(case, case["batch"])
        n = _rows(case, lens)
        seen = n * lens - (n * (n - 1) // 2 if case["causal"] else 0)
        row = case["kv_heads"] * case["head_dim"]
        blocks = int((-(-lens // case["block_size"])).sum())
        return {"bytes": int(lens.sum()) * 2 * row + blocks * (8 * case["kv_heads"] + 4)
                + 2 * int(n.sum()) * case["heads"] * case["head_dim"] * e,
                "flops": 4 * case["heads"] * case["head_dim"] * int(seen.sum())}
    if case["kind"] == "fork":
        lens = _lens(case, case["prompts"])
        part = int((lens % case["block_size"] > 0).sum()) * case["ways"]
        entries = int((-(-lens // case["block_size"])).sum()) * case["ways"]
        return {"bytes": 2 * part * _block_bytes(case) + 20 * entries, "flops": entries}
    if case["kind"] == "compact":
        n = _pool_rows(case)
        used = int(n.sum()) - int(n[0::2].sum() + n[1::2].sum()) // 2
        moved = used * (case["blocks"] - used) // case["blocks"]
        return {"bytes": 2 * moved * _block_bytes(case) + 20 * case["blocks"], "flops": case["blocks"]}
    rows = case["batch"] * (case["drafts"] + 1)
    lists = case["batch"] * (case["prompt"] + case["generated"]) // 2 + 2 * case["batch"] * case["biases"]
    touched = (case["batch"] * (case["drafts"] + 1) * (min(case["prompt"], 64) + case["generated"] // 2)
               if case["penalties"] else 0) + rows * case["biases"]
    masked = rows * case["vocab"] if case["masks"] else 0
    return {"bytes": 4 * lists + 2 * e * touched + masked // 8 + int(masked * (1 - case["allowed"])) * e,
            "flops": 4 * touched + masked}


# ---- inputs -----------------------------------------------------------------------------


def _tables(rng, need, nb):
    """Block tables of rows of these block counts over shuffled blocks 1.., and the ids left."""
    ids = rng.permutation(np.arange(1, nb)).astype(np.uint32)
    t = np.zeros((len(need), int(need.max())), np.uint32)
    at = np.concatenate([[0], np.cumsum(need)])
    for s in range(len(need)):
        t[s, :need[s]] = ids[at[s]:at[s + 1]]
    return t, ids[at[-1]:]


def _scaled_cache(case, nb, gen, dev):
    """One layer's K and V in 8 bits with their scales; amplitudes vary from block to block."""
    d, bs, kvh = case["head_dim"], case["block_size"], case["kv_heads"]
    out = []
    for shape in ((nb, kvh, d // 16, bs, 16), (nb, kvh, d, bs)):
        amp = torch.empty((nb, kvh), device=dev).normal_(generator=gen).mul_(0.5).exp_()
        scale = torch.exp2(torch.ceil(torch.log2(amp * (4.5 / _TOP))))
        if not case.get("pow2", True):
            scale = scale * torch.empty((nb, kvh), device=dev).uniform_(0.6, 1.0, generator=gen)
        lead = (nb, kvh) + (1,) * (len(shape) - 2)
        x = torch.empty(shape, device=dev).normal_(generator=gen).mul_((amp / scale).view(lead))
        out += [x.clamp_(-_TOP, _TOP).to(torch.float8_e4m3fn), scale]
    return out  # kc, ks, vc, vs


def _u32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.uint32)).to(dev)


def _prepare_pages(s, case, rng, gen, dev):
    d, bs, kvh = case["head_dim"], case["block_size"], case["kv_heads"]
    if case["kind"] == "fork":
        lens = _lens(case, case["prompts"])
        need = -(-lens // bs)
        nb = int(need.sum()) + case["prompts"] * case["ways"] + 1 + int(need.sum()) // 8
        rows = case["prompts"] * (1 + case["ways"])
    else:
        need, nb, rows = _pool_rows(case), case["blocks"], case["rows"]
        lens = need * bs
    t, left = _tables(rng, need, nb)
    cols = int(need.max()) + 2
    tables = np.zeros((rows, cols), np.uint32)
    tables[:len(need), :t.shape[1]] = t
    held, at = np.zeros(rows, np.uint32), np.zeros(rows, np.uint32)
    held[:len(need)], at[:len(need)] = need, lens
    ring = np.zeros(nb, np.uint32)
    ring[:len(left)] = left
    s.update(nb=nb, tables=_u32(tables, dev), held=_u32(held, dev), positions=_u32(at, dev),
             ring=_u32(ring, dev), state=_u32([0, len(left)], dev),
             shared=torch.zeros(nb, dtype=torch.int32, device=dev).view(torch.uint32))
    # a tensor for all layers' K, V and scales each; the layers' parts are what is copied
    s["pools"] = {}
    for name, shape in (("key", (kvh, d // 16, bs, 16)), ("value", (kvh, d, bs))):
        shape = (case["layers"], nb) + shape
        if case["scaled"]:
            b = torch.randint(0, 254, shape, dtype=torch.uint8, generator=gen, device=dev)
            b += b >= 127  # no NaN
            s["pools"][name + "_cache"] = b.view(torch.float8_e4m3fn)
            s["pools"][name + "_scales"] = torch.empty(shape[:3], device=dev).uniform_(
                0.001, 0.1, generator=gen)
        else:
            b = torch.empty(shape, dtype=torch.bfloat16, device=dev).normal_(generator=gen)
            s["pools"][name + "_cache"] = b if name == "value" else b.view(
                shape[:3] + (d // 8, bs, 8))
    s["buffers"] = [layer for pool in s["pools"].values() for layer in pool]
    if case["kind"] == "fork":
        n, ways = case["prompts"], case["ways"]
        s["src"] = _u32(np.repeat(np.arange(n), ways), dev)
        s["dst"] = _u32(n + np.arange(n * ways), dev)
        s["keep"] = _u32(np.where(np.arange(rows) < n, cols, 0), dev)
    else:
        # the even rows end in one pass, the odd ones in the next
        odd = np.arange(rows) % 2
        s["keep"] = [_u32(np.where(odd == turn, 0, cols), dev) for turn in (0, 1)]
        s["target"], s["turn"] = _u32(lens, dev), 0
    if own:
        a = s["alloc"] = _vpa().DeviceBlockAllocator(nb, bs, rows, cols, dev)
        a.block_tables, a.row_blocks, a.positions = s["tables"], s["held"], s["positions"]
        a.free_ring, a.free_ring_state, a.shared = s["ring"], s["state"], s["shared"]


def _prepare_logits(s, case, rng, gen, dev):
    b, k, v = case["batch"], case["drafts"], case["vocab"]
    s["logits"] = torch.empty((b, k + 1, v), device=dev).normal_(generator=gen).mul_(2.5).to(
        _TORCH[case["dtype"]])
    # text repeats its common words; a recording's prompt is mostly one placeholder

    def text(n):
        return np.minimum((v * rng.random((b, n)) ** 6).astype(np.int64), v - 1)

    cap = case["generated"] + 32
    s["generated"] = _u32(text(cap), dev)
    s["gen_len"] = _u32(rng.integers(case["generated"] // 2, case["generated"], size=b,
                                     endpoint=True), dev)
    s["prompt"] = s["prompt_len"] = s["drafts"] = s["bias_ids"] = s["allowed"] = None
    s["rep"] = s["pres"] = s["freq"] = s["bias"] = s["bias_len"] = s["which"] = None
    if case["prompt"]:
        p = text(case["prompt"])
        p[:, min(30, case["prompt"]):] = v // 2
        s["prompt"] = _u32(p, dev)
        s["prompt_len"] = _u32(rng.integers((case["prompt"] + 1) // 2, case["prompt"], size=b,
                                            endpoint=True), dev)
    if k:
        s["drafts"] = _u32(text(k), dev)
    if case["penalties"]:
        for name, lo, hi in (("rep", 1.0, 1.3), ("pres", 0.0, 0.6), ("freq", 0.0, 0.4)):
            s[name] = torch.empty(b, device=dev).uniform_(lo, hi, generator=gen)
    n = min(case["biases"], v)
    if n:
        ids = np.stack([rng.permutation(min(v, 4 * n))[:n] * (v // min(v, 4 * n)) for _ in range(b)])
        s["bias_ids"] = _u32(ids, dev)
        s["bias"] = torch.empty((b, n), device=dev).uniform_(-5, 5, generator=gen)
        s["bias_len"] = _u32(rng.integers(0, n, size=b, endpoint=True), dev)
    if case["masks"]:
        words = -(-v // 32)
        bits = torch.rand((case["masks"], words, 32), generator=gen, device=dev) < case["allowed"]
        weight = torch.tensor([1 << i for i in range(31)] + [-(1 << 31)], device=dev)
        s["allowed"] = (bits * weight).sum(-1).to(torch.int32).view(torch.uint32)
        which = rng.integers(0, case["masks"], size=(b, k + 1))
        s["which"] = _u32(np.where(rng.random((b, k + 1)) < 0.9, which, _NONE), dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    s = {"case": case}
    if case["kind"] == "logits":
        _prepare_logits(s, case, rng, gen, dev)
        return s
    if case["kind"] in ("fork", "compact"):
        _prepare_pages(s, case, rng, gen, dev)
        return s
    dt, bs, kvh, d = _TORCH[case["dtype"]], case["block_size"], case["kv_heads"], case["head_dim"]

    def rand(*shape):
        return torch.empty(shape, dtype=dt, device=dev).normal_(generator=gen)

    if case["kind"] == "append":
        t = case["tokens"]
        prior, lens = _runs(case)
    else:
        lens = _lens(case, case["batch"])
    need = -(-lens // bs)
    nb = int(need.sum()) + 1 + int(need.sum()) // 8
    tables, _ = _tables(rng, need, nb)
    s["kc"], s["ks"], s["vc"], s["vs"] = _scaled_cache(case, nb, gen, dev)
    if case["kind"] == "append":
        # rows of one projection's output, louder from token to token
        kv = rand(t, 2 * kvh * d) * torch.empty((t, 1), dtype=dt, device=dev).uniform_(
            0.5, 2.0, generator=gen)
        s["k"] = kv[:, :kvh * d].view(t, kvh, d)
        s["v"] = kv[:, kvh * d:].view(t, kvh, d)
        which = np.arange(t) // case["run_len"]
        pos = prior[which] + np.arange(t) % case["run_len"]
        s["slots"] = torch.from_numpy(tables[which, pos // bs].astype(np.int64) * bs + pos % bs).to(dev)
        return s
    n = _rows(case, lens)
    s["tables"], s["lens"], s["max_len"] = _u32(tables, dev), _u32(lens, dev), int(lens.max())
    s["max_rows"] = int(n.max())
    s["cu"] = None if case["rows"] == 1 else _u32(np.concatenate([[0], np.cumsum(n)]), dev)
    s["q"] = rand(int(n.sum()), case["heads"], d)
    return s


# ---- one pass ---------------------------------------------------------------------------


def run(s):
    kind = s["case"]["kind"]
    if own:
        return _run_own(_vpa(), s, kind)
    return _PLAIN[kind](s)


def _pages(s):
    out = {name: s[name].view(torch.int32) for name in ("tables", "held", "positions", "ring",
                                                         "state", "shared")}
    return {**out, **s["pools"]}


def _run_own(vpa, s, kind):
    case = s["case"]
    if kind == "append":
        vpa.reshape_and_cache_block_scaled(s["k"], s["v"], s["ks"], s["vs"], s["kc"], s["vc"], s["slots"])
        return {"key_cache": s["kc"], "value_cache": s["vc"], "key_scales": s["ks"],
                "value_scales": s["vs"]}
    if kind == "attention":
        return vpa.paged_attention_block_scaled(
            s["q"], s["ks"], s["vs"], s["kc"], s["vc"], s["tables"], s["lens"],
            case["head_dim"] ** -0.5, cu_seqlens_q=s["cu"], causal=case["causal"],
            max_query_len=s["max_rows"], max_context_len=s["max_len"])
    if kind == "fork":
        ok = s["alloc"].fork(s["src"], s["dst"], s["buffers"])
        s["alloc"].release(s["keep"])
        return {"ok": ok, **_pages(s)}
    if kind == "compact":
        s["alloc"].release(s["keep"][s["turn"]])
        s["turn"] ^= 1
        src, dst, count = s["alloc"].compact(s["buffers"])
        s["alloc"].allocate(s["target"])
        return {"moved": count.view(torch.int32), **_pages(s)}
    vpa.adjust_logits(s["logits"], s["generated"], s["gen_len"], prompt=s["prompt"],
                      prompt_len=s["prompt_len"], draft_ids=s["drafts"], repetition=s["rep"],
                      presence=s["pres"], frequency=s["freq"], bias_ids=s["bias_ids"],
                      bias=s["bias"], bias_len=s["bias_len"], allowed=s["allowed"],
                      allowed_rows=s["which"])
    return s["logits"]


def _needed_scale(amax):
    """The smallest power of two s with amax <= 448 s."""
    m, e = torch.frexp(amax.float())  # amax = m 2^e, m in [0.5, 1)
    exp = torch.where(m <= 0.875, e - 9, e - 8)  # 448 = 0.875 2^9
    exp = torch.where(amax > 0, exp, _LEAST).clamp_(min=_LEAST)
    return torch.ldexp(torch.ones_like(m), exp)


def _plain_append(s):
    bs = s["case"]["block_size"]
    slots = s["slots"]
    blk, off = slots // bs, slots % bs
    t, kvh, d = s["k"].shape
    touched, place = torch.unique(blk, return_inverse=True)
    fresh = torch.zeros(len(touched), device=slots.device, dtype=torch.bool).index_put_(
        (place,), off == 0, accumulate=True)
    for x, cache, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        x = x.float()
        amax = torch.zeros((len(touched), kvh), device=x.device).index_reduce_(
            0, place, x.abs().amax(-1), "amax")
        old = scales[touched]
        new = torch.where(fresh[:, None], _needed_scale(amax), torch.maximum(old, _needed_scale(amax)))
        grown = (~fresh[:, None] & (new > old)).view(-1, kvh, *(1,) * (cache.dim() - 2))
        ratio = (old / new).view_as(grown)
        bytes_ = cache.view(torch.uint8)
        held = bytes_[touched].view(torch.float8_e4m3fn)
        again = (held.float() * ratio).to(torch.float8_e4m3fn).view(torch.uint8)
        bytes_[touched] = torch.where(grown, again, held.view(torch.uint8))
        scales[touched] = new
        y = (x / scales[blk][..., None]).clamp(-_TOP, _TOP).to(torch.float8_e4m3fn).view(torch.uint8)
        if cache.dim() == 5:
            y = y.view(t, kvh, d // 16, 16)
        bytes_[blk, :, :, off] = y
    return {"key_cache": s["kc"], "value_cache": s["vc"], "key_scales": s["ks"],
            "value_scales": s["vs"]}


def _plain_attention(s):
    case = s["case"]
    kvh, d, n_max, l_max = case["kv_heads"], case["head_dim"], s["max_rows"], s["max_len"]
    group = case["heads"] // kvh
    dev = s["q"].device
    lens = s["lens"].view(torch.int32).long()
    b = lens.shape[0]
    cu = torch.arange(b + 1, device=dev) if s["cu"] is None else s["cu"].view(torch.int32).long()
    ids = s["tables"].view(torch.int32).long()
    k = s["kc"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).float()  # [b, cols, kvh, d/x, bs, x]
    k = (k * s["ks"][ids][..., None, None, None]).permute(0, 2, 3, 5, 1, 4)
    k = k.reshape(b, kvh, d, -1)[..., :l_max].contiguous()
    v = s["vc"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).float()  # [b, cols, kvh, d, bs]
    v = (v * s["vs"][ids][..., None, None]).permute(0, 2, 1, 4, 3)
    v = v.reshape(b, kvh, -1, d)[:, :, :l_max].contiguous()
    row = torch.arange(n_max, device=dev)
    n = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + row).clamp_(max=s["q"].shape[0] - 1)
    q = s["q"][at].float().reshape(b, n_max, kvh, group, d).permute(0, 2, 3, 1, 4)
    logits = torch.matmul(q.reshape(b, kvh, group * n_max, d), k) * d ** -0.5
    logits = logits.view(b, kvh, group, n_max, l_max)
    tok = torch.arange(l_max, device=dev)
    last = row[None] + (lens - n)[:, None] if case["causal"] else lens[:, None].expand(b, n_max) - 1
    seen = (tok[None, None] <= last[..., None])[:, None, None]
    logits.masked_fill_(~seen, -math.inf)
    p = torch.exp_(logits.sub_(logits.amax(-1, keepdim=True)))
    total = p.sum(-1, keepdim=True) + (0.0 if case["causal"] and s["cu"] is not None else 1e-6)
    o = torch.matmul(p.view(b, kvh, group * n_max, l_max), v).view(b, kvh, group, n_max, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(b, n_max, case["heads"], d)
    return o[row[None] < n[:, None]].to(s["q"].dtype)


def _plain_copy(s, src, dst):
    for x in s["buffers"]:
        if x.element_size() == 1:  # bytes are indexed as bytes
            x = x.view(torch.uint8)
        x[dst] = x[src]


def _plain_release(s, keep):
    """Rows in order give blocks back, last block first; one that others hold stays theirs."""
    tables, held, shared, ring, state = (s[n].view(torch.int32) for n in (
        "tables", "held", "shared", "ring", "state"))
    rows, cols = tables.shape
    col = torch.arange(cols - 1, -1, -1, device=tables.device)
    keep = keep.view(torch.int32)
    gone = (col >= keep[:, None]) & (col < held[:, None])
    ids = tables.flip(1)[gone].long()
    ids = ids[ids != 0]
    given = torch.zeros(s["nb"], dtype=torch.int32, device=ids.device).index_add_(
        0, ids, torch.ones_like(ids, dtype=torch.int32))
    free = given > shared
    place = torch.arange(len(ids), device=ids.device)
    last = torch.zeros(s["nb"], dtype=torch.int64, device=ids.device).index_reduce_(
        0, ids, place, "amax")
    back = ids[free[ids] & (last[ids] == place)]
    at = (state[0] + state[1] + torch.arange(len(back), device=ids.device)) % s["nb"]
    ring[at] = back.to(torch.int32)
    state[1] += len(back)
    shared.copy_(torch.where(free, 0, shared - given))
    held.copy_(torch.minimum(held, keep))


def _plain_fork(s):
    bs = s["case"]["block_size"]
    tables, held, at, shared, ring, state = (s[n].view(torch.int32) for n in (
        "tables", "held", "positions", "shared", "ring", "state"))
    src, dst = s["src"].view(torch.int32).long(), s["dst"].view(torch.int32).long()
    tokens = torch.minimum(at[src], held[src] * bs)
    full, part = tokens // bs, tokens % bs > 0
    rank = part.cumsum(0) - part.long()
    ok = (held[dst] == 0) & (~part | (rank < state[1]))
    new = ring[(state[0] + rank) % s["nb"]]
    col = torch.arange(tables.shape[1], device=src.device)
    old = tables[src]
    whole = col < full[:, None]
    row = torch.where(whole, old, tables[dst])
    row = torch.where(part[:, None] & (col == full[:, None]), new[:, None], row)
    tables[dst] = row
    ids = old[whole].long()
    shared.index_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))
    held[dst] = full + part.to(torch.int32)
    at[dst] = tokens
    used = part.sum().to(torch.int32)
    state[0] = (state[0] + used) % s["nb"]
    state[1] -= used
    _plain_copy(s, old.gather(1, full.long().clamp(max=len(col) - 1)[:, None])[part, 0].long(),
                new[part].long())
    _plain_release(s, s["keep"])
    return {"ok": ok.to(torch.uint8), **_pages(s)}


def _plain_compact(s):
    nb, bs = s["nb"], s["case"]["block_size"]
    tables, held, shared, ring, state = (s[n].view(torch.int32) for n in (
        "tables", "held", "shared", "ring", "state"))
    dev = tables.device
    _plain_release(s, s["keep"][s["turn"]])
    s["turn"] ^= 1
    # the k-th block in use past the front takes the k-th free place in it
    turn = torch.arange(nb, device=dev)
    free = torch.zeros(nb, dtype=torch.bool, device=dev)
    free[ring[(state[0] + turn) % nb][turn < state[1]].long()] = True
    n_free = free.sum()
    front = nb - 1 - n_free
    place = turn[1:]
    src, dst = place[~free[1:] & (place > front)], place[free[1:] & (place <= front)]
    to = turn.clone()
    to[src] = dst
    col = torch.arange(tables.shape[1], device=dev)
    tables.copy_(torch.where(col < held[:, None], to[tables.long()].to(torch.int32), tables))
    shared[dst] = shared[src]
    shared[src] = 0
    ring.copy_(torch.where(turn < n_free, front + 1 + turn, ring.long()).to(torch.int32))
    state[0], state[1] = 0, n_free
    _plain_copy(s, src, dst)
    # rows that ended start again, from the front of the free ones
    need = -(-s["target"].view(torch.int32) // bs)
    more = need - held
    want = (col >= held[:, None]) & (col < need[:, None])
    tables[want] = ring[(state[0] + torch.arange(int(more.sum()), device=dev)) % nb]
    state[0] = (state[0] + more.sum()) % nb
    state[1] -= more.sum()
    held.copy_(need)
    return {"moved": torch.tensor([len(src)], dtype=torch.int32, device=dev), **_pages(s)}


def _plain_logits(s):
    case = s["case"]
    b, k, v = case["batch"], case["drafts"], case["vocab"]
    dev = s["logits"].device
    x = s["logits"].float()

    def ids(t):
        return t.view(torch.int32).long()

    def times(list_, length):
        inside = torch.arange(list_.shape[1], device=dev) < ids(length)[:, None]
        return torch.zeros((b, v), device=dev).scatter_add_(1, ids(list_), inside.float())

    if case["penalties"]:
        count = times(s["generated"], s["gen_len"])[:, None].repeat(1, k + 1, 1)
        for i in range(k):
            one = torch.ones((b, 1, 1), device=dev).expand(b, k - i, 1)
            count[:, i + 1:].scatter_add_(2, ids(s["drafts"])[:, None, i:i + 1].expand(b, k - i, 1), one)
        seen = count > 0
        if s["prompt"] is not None:
            seen = seen | (times(s["prompt"], s["prompt_len"]) > 0)[:, None]
        rep, pres, freq = (s[n][:, None, None] for n in ("rep", "pres", "freq"))
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        x = x - freq * count - pres * (count > 0)
    if s["bias"] is not None:
        inside = torch.arange(s["bias"].shape[1], device=dev) < ids(s["bias_len"])[:, None]
        x = x + torch.zeros((b, v), device=dev).scatter_add_(
            1, ids(s["bias_ids"]), s["bias"] * inside)[:, None]
    if s["allowed"] is not None:
        tok = torch.arange(v, device=dev)
        words = ids(s["allowed"])[:, tok // 32]
        free = (words >> (tok % 32)) & 1
        which = ids(s["which"])
        x = torch.where((free[which.clamp(min=0)] == 1) | (which < 0)[..., None], x, -math.inf)
    s["logits"].copy_(x)
    return s["logits"]


_PLAIN = {"append": _plain_append, "attention": _plain_attention, "fork": _plain_fork,
          "compact": _plain_compact, "logits": _plain_logits}


# ---- the definitions in 64 bits -----------------------------------------------------------


def _exact_append(case, s):
    bs, d = case["block_size"], case["head_dim"]
    slot = s["slots"].cpu().numpy()
    blocks = {}
    for t, at in enumerate(slot):
        blocks.setdefault(int(at) // bs, []).append(t)
    own_block = torch.from_numpy(slot // bs).to("cuda")
    first = torch.tensor([min(int(slot[t]) % bs for t in ts) == 0 for ts in blocks.values()],
                         device="cuda")[:, None]
    ids = torch.tensor(list(blocks), device="cuda")
    spot = {blk: i for i, blk in enumerate(blocks)}
    at = torch.tensor([spot[int(x) // bs] for x in slot], device="cuda")
    out = {}
    for name, x, cache, scales in (("key", s["k"], s["kc"], s["ks"]), ("value", s["v"], s["vc"], s["vs"])):
        x = x.double()
        top = torch.full((len(ids), x.shape[1]), 2.0 ** _LEAST * _TOP, dtype=torch.float64, device="cuda")
        top.scatter_reduce_(0, at[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
        want = torch.pow(2.0, torch.ceil(torch.log2(top) - math.log2(_TOP) - 1e-12))
        was = scales[ids].double()
        new = torch.where(first | (want > was), want, was)
        y, sc = cache.double(), scales.double()
        keep = torch.where(first, 1.0, was / new)
        y[ids] *= keep.view(keep.shape + (1,) * (y.dim() - 2))
        sc[ids] = new
        z = x / sc[own_block][..., None]
        if name == "key":
            z = z.reshape(z.shape[0], z.shape[1], d // 16, 16)
        y[slot // bs, :, :, slot % bs] = z
        out[name + "_cache"], out[name + "_scales"] = y, sc
    return out


def _exact_attention(case, s):
    lens = _lens(case, case["batch"])
    n = _rows(case, lens)
    kvh, bs, d = case["kv_heads"], case["block_size"], case["head_dim"]
    group = case["heads"] // kvh
    tables = s["tables"].view(torch.int32).long()
    eps = 0.0 if case["causal"] and s["cu"] is not None else 1e-6
    out, a = [], 0
    for i in range(len(lens)):
        size, rows = int(lens[i]), int(n[i])
        ids = tables[i, :-(-size // bs)]
        k = s["kc"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
        k = k * s["ks"][ids].double()[:, :, None, None, None]
        k = k.permute(1, 2, 4, 0, 3).reshape(kvh, d, -1)[..., :size].contiguous()
        v = s["vc"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
        v = v * s["vs"][ids].double()[:, :, None, None]
        v = v.permute(1, 0, 3, 2).reshape(kvh, -1, d)[:, :size].contiguous()
        q = s["q"][a:a + rows].double().reshape(rows, kvh, group, d).permute(1, 0, 2, 3)
        a += rows
        z = torch.bmm(q.reshape(kvh, rows * group, d), k) / math.sqrt(d)
        if case["causal"]:
            see = size - rows + 1 + torch.arange(rows, device=z.device).repeat_interleave(group)
            z = z.masked_fill(torch.arange(size, device=z.device) >= see[:, None], -math.inf)
        top = z.amax(-1, keepdim=True)
        p = torch.exp(z - top)
        o = torch.bmm(p, v) / (p.sum(-1, keepdim=True) + eps)
        out.append(o.reshape(kvh, rows, group, d).permute(1, 0, 2, 3).reshape(rows, -1, d))
    return torch.cat(out)


def _exact_logits(case, s):
    x = s["logits"].double().cpu().numpy()
    lists = {n: None if s[n] is None else s[n].cpu().numpy() for n in (
        "generated", "gen_len", "prompt", "prompt_len", "drafts", "rep", "pres", "freq", "bias_ids",
        "bias", "bias_len", "allowed", "which")}
    v = case["vocab"]
    for r in range(case["batch"]):
        told = lists["generated"][r, :lists["gen_len"][r]].astype(np.int64)
        asked = np.zeros(0, np.int64) if lists["prompt"] is None else \
            np.unique(lists["prompt"][r, :lists["prompt_len"][r]].astype(np.int64))
        for i in range(case["drafts"] + 1):
            row = x[r, i]
            if case["penalties"]:
                all_ = np.concatenate([told, lists["drafts"][r, :i].astype(np.int64)]) if i else told
                ids, count = np.unique(all_, return_counts=True)
                once = np.union1d(ids, asked)
                rep = float(lists["rep"][r])
                row[once] = np.where(row[once] > 0, row[once] / rep, row[once] * rep)
                row[ids] -= float(lists["freq"][r]) * count + float(lists["pres"][r])
            if lists["bias"] is not None:
                m = int(lists["bias_len"][r])
                row[lists["bias_ids"][r, :m]] += lists["bias"][r, :m]
            if lists["allowed"] is not None and lists["which"][r, i] != _NONE:
                bits = np.unpackbits(lists["allowed"][lists["which"][r, i]].view(np.uint8),
                                     bitorder="little")[:v]
                row[bits == 0] = -np.inf
    return torch.from_numpy(x).to("cuda")


def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return None  # whole numbers and copies
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "logits": _exact_logits}[
        case["kind"]](case, s)
