"""Plain 64-bit restatements of the decode loop's operators (rotary rows,
attention weights, eviction, draft verification), from their definitions, for
the tests. numpy only; caches in the paged layout as float64."""

import numpy as np


def rotary(x, positions, inv_freq, axes, *, weight=None, eps=1e-6, adjacent=False):
    """x [T, H, D] -> (y [T, H, D], scale of each value's rounding)."""
    x = x.astype(np.float64)
    d, half = x.shape[2], len(inv_freq)
    if weight is not None:
        x = x * weight.astype(np.float64) / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps)
    a = np.arange(half) * 2 if adjacent else np.arange(half)
    b = a + 1 if adjacent else a + half
    pos = np.atleast_2d(positions).astype(np.float64)
    axes = np.minimum(np.zeros(half, int) if axes is None else axes, len(pos) - 1)
    angle = (pos[axes] * np.asarray(inv_freq, np.float64)[:, None]).T[:, None, :]
    y, mag = x.copy(), np.abs(x)
    y[..., a] = x[..., a] * np.cos(angle) - x[..., b] * np.sin(angle)
    y[..., b] = x[..., b] * np.cos(angle) + x[..., a] * np.sin(angle)
    mag[..., a] = mag[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    assert y.shape[2] == d
    return y, mag


def rows_of(cache, table, length):
    """K or V rows [KVH, length, D] of one sequence from a float64 cache."""
    bs = cache.shape[3]
    t = np.arange(length)
    rows = cache[table[t // bs].astype(np.int64), :, :, t % bs]  # [length, KVH, D / x, x] or [.., D]
    return rows.reshape(length, cache.shape[1], -1).transpose(1, 0, 2)


def attention_weights(q, key_cache, tables, lens, scale, scores, cu=None, causal=True):
    """scores + the softmax weights of q's rows; absent blocks (ids past the pool)
    get none."""
    out = scores.astype(np.float64)
    q = q.astype(np.float64)
    nb, kvh, _, bs, _ = key_cache.shape
    group = q.shape[1] // kvh
    cu = np.arange(len(lens) + 1) if cu is None else np.asarray(cu, np.int64)
    for s, size in enumerate(lens):
        size = int(size)
        n = int(cu[s + 1] - cu[s])
        if size == 0 or n == 0:
            continue
        table = tables[s].astype(np.int64)
        there = table[np.arange(size) // bs] < nb
        k = rows_of(key_cache, np.where(table < nb, table, 0), size)
        for r in range(n):
            see = there & (np.arange(size) <= (r + size - n if causal else size))
            if not see.any():
                continue
            for h in range(q.shape[1]):
                logit = np.where(see, scale * (k[h // group] @ q[cu[s] + r, h]), -np.inf)
                with np.errstate(invalid="ignore"):
                    p = np.where(see, np.exp(logit - logit[see].max()), 0.0)
                out[s, h // group, :size] += p / p.sum()
    return out


def evict(scores, lens, budget, first, last):
    """(new lens, kept [B][KVH] index arrays)."""
    b, kvh, _ = scores.shape
    kept = [[None] * kvh for _ in range(b)]
    for s in range(b):
        size = int(lens[s])
        for j in range(kvh):
            if size <= budget:
                kept[s][j] = np.arange(size)
                continue
            lo, hi = first, size - last
            mid = scores[s, j, lo:hi].astype(np.float64)
            # NaN below every number, equal scores by place
            order = sorted(range(hi - lo), key=lambda t: (np.isnan(mid[t]), -mid[t] if not
                                                          np.isnan(mid[t]) else 0.0, t))
            keep = list(range(lo)) + [lo + t for t in order[:budget - first - last]] + \
                list(range(hi, size))
            kept[s][j] = np.array(sorted(keep), dtype=np.int64)
    return np.minimum(lens, budget).astype(np.uint32), kept


def moved(cache, tables, kept, is_key):
    """The cache (any dtype) with each head's kept tokens at the front."""
    out = cache.copy()
    bs = cache.shape[3]
    for s, heads in enumerate(kept):
        for j, keep in enumerate(heads):
            to = np.arange(len(keep))
            sb, so = tables[s][keep // bs].astype(np.int64), keep % bs
            db, do = tables[s][to // bs].astype(np.int64), to % bs
            if is_key:
                out[db, j, :, do] = cache[sb, j, :, so]
            else:
                out[db, j, :, do] = cache[sb, j, :, so]
    return out


def softmax(row, temperature):
    row = row.astype(np.float64)
    ok = ~np.isnan(row) & (row != -np.inf)
    p = np.zeros(row.shape)
    if ok.any():
        top = row[ok].max()
        with np.errstate(invalid="ignore", over="ignore"):
            e = np.exp((row[ok] - top) / temperature)
        p[ok] = np.where(row[ok] == top, 1.0, np.nan_to_num(e, nan=0.0))
        p /= p.sum()
    return p


def draw(r, u):
    up = np.cumsum(r)
    if not up[-1] > 0:
        return None
    hit = np.nonzero(up > u * up[-1])[0]
    return int(hit[0]) if len(hit) else int(np.nonzero(r > 0)[0][-1])


def verify(target, draft_ids, accept_u, sample_u, draft=None, num_drafts=None, temperature=None):
    """(ids [B, K + 1] with 0xffffffff behind, count [B], margins [B]: the smallest
    relative distance of a decision from its border)."""
    b, k1, v = target.shape
    ids = np.full((b, k1), 0xFFFFFFFF, np.uint32)
    count = np.zeros(b, np.uint32)
    margin = np.full(b, np.inf)
    for s in range(b):
        n = k1 - 1 if num_drafts is None else min(int(num_drafts[s]), k1 - 1)
        t = 1.0 if temperature is None else float(temperature[s])
        greedy = not t > 0
        took, last = 0, None
        while True:
            row = target[s, took].astype(np.float64)
            if greedy:
                last = int(np.argmax(np.where(np.isnan(row), -np.inf, row)))
            p = None if greedy else softmax(row, t)
            if took == n:
                break
            x = int(draft_ids[s, took])
            if greedy:
                if x != last:
                    break
            else:
                q = None if draft is None else softmax(draft[s, took], t)
                px = p[x] if x < v else 0.0
                have = float(accept_u[s, took]) * (1.0 if q is None else (q[x] if x < v else 1.0))
                if max(px, have) > 0:  # (0 and 0 are exact: masked logits weigh exactly 0)
                    margin[s] = min(margin[s], abs(have - px) / max(px, have))
                if not have < px:
                    if q is None:
                        r = p.copy()
                        if x < v:
                            r[x] = 0
                    else:
                        r = np.maximum(p - q, 0)
                        if not r.sum() > 0:
                            r = p
                    last = draw(r, float(sample_u[s]))
                    if last is None:  # p is all at x, or nowhere
                        last = x if x < v and p[x] > 0 else 0
                    break
            ids[s, took] = x
            took += 1
        if last is None:
            last = draw(p, float(sample_u[s]))
            last = 0 if last is None else last
        ids[s, took] = last
        count[s] = took + 1
    return ids, count, margin
