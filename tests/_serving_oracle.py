"""Plain restatements, for the tests, of the block-scaled cache, of rows that share
blocks and of adjusted logits: in 64 bits or in whole numbers, one element, block or
row after the other, from their definitions. numpy only."""

import math

import numpy as np

from oracle import oracle as orc

TOP = 448.0
NONE = 0xFFFFFFFF


# ---- block-scaled cache -------------------------------------------------------


def e4m3(x):
    """The nearest E4M3 byte (ties to even, saturated, NaN kept)."""
    return orc.fp8_from_f32(np.ascontiguousarray(x, np.float32))


def e4m3_value(b):
    b = np.asarray(b).astype(np.int64)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b & 128, -v, v)


def needed_scale(rows):
    a = np.abs(rows[np.isfinite(rows)])
    if a.size == 0 or a.max() == 0:
        return 2.0 ** -100
    m, e = math.frexp(float(a.max()))  # m 2^e, m in [0.5, 1); 448 = 0.875 2^9
    return 2.0 ** max(-100, e - 9 + (m > 0.875))


def append(key, value, ks, vs, kc, vc, slots):
    """In place, one block of the call and head after the other. Rows f32 [T, KVH, D],
    caches of bytes."""
    nb, kvh, _, bs, x = kc.shape
    runs = []
    for t, slot in enumerate(slots):
        b = int(slot) // bs if 0 <= slot < nb * bs else -1
        if b >= 0 and runs and runs[-1][0] == b and t > 0 and slots[t - 1] >= 0 and \
                int(slots[t - 1]) // bs == b:
            runs[-1][1].append(t)
        elif b >= 0:
            runs.append((b, [t]))
    for b, tokens in runs:
        last = {int(slots[t]) % bs: t for t in tokens}
        for j in range(kvh):
            for rows, scales, cache in ((key, ks, kc), (value, vs, vc)):
                need = needed_scale(np.stack([rows[t, j] for t in last.values()]))
                old = float(scales[b, j])
                tile = cache[b, j]
                if 0 in last:
                    new = need
                else:
                    new = max(old, need)
                    if new > old:
                        tile[...] = e4m3(e4m3_value(tile) * (old / new))
                scales[b, j] = new
                for off, t in last.items():
                    with np.errstate(over="ignore"):
                        q = e4m3(rows[t, j].astype(np.float64) / new)
                    if cache.ndim == 5:
                        tile[:, off, :] = q.reshape(-1, x)
                    else:
                        tile[:, off] = q


def attention(q, ks, vs, kc, vc, tables, lens, scale, cu=None, causal=True, eps=0.0):
    """(out, sum of p |V| / sum of p, largest |scale ks q.K| with absolute products, largest
    vs / sum of p) per row, in 64 bits."""
    nb, kvh, _, bs, _ = kc.shape
    rows, heads, d = q.shape
    group = heads // kvh
    cu = np.arange(len(lens) + 1) if cu is None else np.asarray(cu, np.int64)
    out, mag, prod, low = (np.zeros((rows, heads, n)) for n in (d, d, 1, 1))
    for s, size in enumerate(lens):
        size, n = int(size), int(cu[s + 1] - cu[s])
        if size == 0:
            continue
        t = np.arange(size)
        ids = tables[s][t // bs].astype(np.int64)
        there = ids < nb
        ids = np.where(there, ids, 0)
        k = e4m3_value(kc[ids, :, :, t % bs].reshape(size, kvh, d)) * ks[ids][:, :, None].astype(np.float64)
        v = e4m3_value(vc[ids, :, :, t % bs]) * vs[ids][:, :, None].astype(np.float64)
        for r in range(n):
            see = there & ((t <= r + size - n) if causal else True)
            if not see.any():
                continue
            for h in range(heads):
                j = h // group
                x = q[cu[s] + r, h].astype(np.float64)
                z = scale * (k[see, j] @ x)
                p = np.exp(z - z.max())
                vr = v[see, j]
                out[cu[s] + r, h] = (p @ vr) / (p.sum() + eps)
                mag[cu[s] + r, h] = (p @ np.abs(vr)) / p.sum()
                prod[cu[s] + r, h] = abs(scale) * (np.abs(k[see, j]) @ np.abs(x)).max()
                low[cu[s] + r, h] = np.abs(vs[ids[see], j].astype(np.float64)).max() / p.sum() * see.sum()
    return out, mag, prod, low


def attention_bound(want, mag, prod, low, d, length, unit):
    """What the kernel's roundings come to. ``unit``: half a step of the query's type.

    * a score is a sum of d exact products in f32, scaled three times: off by at most
      (d + 8) 2^-23 of the sum of its absolute products (2^-23: the matrix
      instructions may truncate); it shifts exp by as much, the sum of exps too;
    * exp2 and the running rescales: 2^-20; sums over `length` tokens in f32;
    * probabilities as f16 (16-bit queries): f16's numbers in [1, 2) are 2^-10 apart, so
      2^-11 of themselves; as two f16 values for f32 queries: 2^-22; below f16's normal range 2^-32 of the largest scale times E4M3's
      largest value per token;
    * the output: half a step of its type.
    """
    p = 2.0 ** -22 if unit < 2.0 ** -20 else 2.0 ** -11
    rel = p + 2 * (d + 8) * 2.0 ** -23 * prod + 2.0 ** -20 + length * 2.0 ** -23
    return mag * rel + low * TOP * 2.0 ** -32 + np.abs(want) * unit + 1e-37


# ---- rows that share blocks ---------------------------------------------------


class Pages:
    """The device allocator's state and operations, one row and block at a time."""

    def __init__(self, num_blocks, block_size, rows, cols):
        self.nb, self.bs, self.cols = num_blocks, block_size, cols
        self.tables = np.zeros((rows, cols), np.uint32)
        self.held = np.zeros(rows, np.uint32)
        self.positions = np.zeros(rows, np.uint32)
        self.shared = np.zeros(num_blocks, np.uint32)
        self.ring = np.zeros(num_blocks, np.uint32)
        self.ring[:num_blocks - 1] = np.arange(1, num_blocks)
        self.head, self.count = 0, num_blocks - 1

    def take(self):
        b = self.ring[self.head % self.nb]
        self.head = (self.head + 1) % self.nb
        self.count -= 1
        return b

    def give(self, b):
        if b == 0:
            return
        if self.shared[b] > 0:
            self.shared[b] -= 1
        else:
            self.ring[(self.head + self.count) % self.nb] = b
            self.count += 1

    def allocate(self, target):
        for r, tokens in enumerate(target):
            need = -(-int(tokens) // self.bs)
            if need <= self.held[r] or need > self.cols or need - self.held[r] > self.count:
                continue
            while self.held[r] < need:
                self.tables[r, self.held[r]] = self.take()
                self.held[r] += 1

    def release(self, keep):
        for r, n in enumerate(keep):
            while self.held[r] > n:
                self.held[r] -= 1
                self.give(self.tables[r, self.held[r]])

    def fork(self, src, dst):
        rows = len(self.held)
        held, positions = self.held.copy(), self.positions.copy()
        ok, pairs, claimed = [], [], set()
        for a, b in zip(src, dst):
            good = a < rows and b < rows and held[min(b, rows - 1)] == 0 and b not in claimed
            claimed.add(b)
            if good:
                tokens = min(int(positions[a]), int(held[a]) * self.bs)
                full, part = tokens // self.bs, tokens % self.bs > 0
                good = not part or self.count > 0
            if good:
                for i in range(full):
                    self.tables[b, i] = self.tables[a, i]
                    if self.tables[a, i]:
                        self.shared[self.tables[a, i]] += 1
                if part:
                    new = self.take()
                    pairs.append((int(self.tables[a, full]), int(new)))
                    self.tables[b, full] = new
                self.held[b], self.positions[b] = full + part, tokens
            ok.append(good)
        return ok, pairs

    def unshare(self):
        ok, pairs = [], []
        for r in range(len(self.held)):
            at, inside = divmod(int(self.positions[r]), self.bs)
            ok.append(True)
            if not inside or at >= self.held[r]:
                continue
            b = self.tables[r, at]
            if b == 0 or self.shared[b] == 0:
                continue
            if self.count == 0:
                ok[-1] = False
                continue
            self.shared[b] -= 1
            self.tables[r, at] = self.take()
            pairs.append((int(b), int(self.tables[r, at])))
        return ok, pairs

    def compact(self):
        free = {int(self.ring[(self.head + i) % self.nb]) for i in range(self.count)}
        front = self.nb - 1 - len(free)
        src = [b for b in range(front + 1, self.nb) if b not in free]
        dst = [b for b in range(1, front + 1) if b in free]
        to = dict(zip(src, dst))
        for r in range(len(self.held)):
            for i in range(self.held[r]):
                self.tables[r, i] = to.get(int(self.tables[r, i]), self.tables[r, i])
        for a, b in to.items():
            self.shared[b], self.shared[a] = self.shared[a], 0
        for i in range(len(free)):
            self.ring[i] = front + 1 + i
        self.head, self.count = 0, len(free)
        return list(zip(src, dst))


# ---- logits -------------------------------------------------------------------


def adjust(x, told, asked=(), rep=None, pres=None, freq=None, bias=(), mask=None):
    """(row, what its roundings are relative to) of one row x in 64 bits; ``told`` and
    ``asked`` are ids, ``bias`` pairs (id, value), ``mask`` truth values or None."""
    y = x.astype(np.float64)
    mag = np.abs(y)
    v = len(y)
    counts = {}
    for t in told:
        if t < v:
            counts[int(t)] = counts.get(int(t), 0) + 1
    with np.errstate(invalid="ignore", over="ignore"):
        if rep is not None:
            for t in set(counts) | {int(t) for t in asked if t < v}:
                y[t] = y[t] / rep if y[t] > 0 else y[t] * rep
        mag = np.maximum(mag, np.abs(y))
        for t, c in counts.items():
            off = (freq or 0.0) * c + (pres or 0.0)
            y[t] -= off
            mag[t] += abs(off)
        for t, b in dict((int(t), b) for t, b in bias).items():
            if t < v:
                y[t] += b
                mag[t] += abs(b)
    if mask is not None:
        y[~mask] = -np.inf
    return y, mag
