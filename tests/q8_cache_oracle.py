"""The int8 key/value cache in numpy: its write as include/accel_b200.h states
it, and attention over it in 64 bits."""

import numpy as np


def tables(context, d, theta=10000.0):
    angle = np.outer(np.arange(context, dtype=np.float64), theta ** (-np.arange(0, d, 2) / d))
    angle = np.concatenate([angle, angle], axis=1)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def rope(x, cos, sin):
    """x [rows, heads, d] fp32, cos and sin [rows, d]: each step rounded."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    cos, sin = cos[:, None], sin[:, None]
    return np.concatenate([a * cos[..., :half] - b * sin[..., :half], b * cos[..., half:] + a * sin[..., half:]], -1)


def scale_for(amax):
    s = np.float32(2.0 ** -126)
    while np.float64(s) * 127 < np.float64(amax):
        s = np.float32(s * 2)
    return s


class Cache:
    def __init__(self, slots, kv, context, d, block):
        self.q = {n: np.zeros((slots, kv, context, d), np.int8) for n in "kv"}
        self.s = {n: np.zeros((slots, kv, -(-context // block)), np.float32) for n in "kv"}
        self.block, self.context = block, context

    def write(self, slot, pos0, new):
        """new {"k", "v"} [rows, kv, d] at positions pos0 + i of a slot."""
        block = self.block
        for name in "kv":
            for g in range(new[name].shape[1]):
                q, s, x = self.q[name][slot, g], self.s[name][slot, g], new[name][:, g]
                for j in range(pos0 // block, (pos0 + len(x) - 1) // block + 1):
                    lo, hi = max(j * block, pos0), min((j + 1) * block, pos0 + len(x))
                    part = x[lo - pos0:hi - pos0]
                    fine = np.abs(part[np.isfinite(part)])
                    amax = fine.max() if fine.size else np.float32(0)
                    held = lo > j * block and np.isfinite(s[j]) and s[j] > 0
                    if not (held and np.float32(127) * s[j] >= amax):
                        now = scale_for(amax)
                        ratio = s[j] / now if held else np.float32(0)
                        old = q[j * block:lo].astype(np.float32) * ratio
                        q[j * block:lo] = np.clip(np.rint(old), -127, 127).astype(np.int8)
                        s[j] = now
                    with np.errstate(invalid="ignore"):
                        y = np.clip(np.rint(part / s[j]), -127, 127)
                    q[lo:hi] = np.where(np.isnan(part), 0, y).astype(np.int8)

    def value(self, name, slot, g, t):
        """Rows t (an index array) of a run in 64 bits."""
        return (self.q[name][slot, g, t].astype(np.float64) *
                self.s[name][slot, g, t // self.block].astype(np.float64)[:, None])


def visible(pos, window, sinks):
    t = np.arange(pos + 1)
    return t[(t > pos - window) | (t < sinks)] if window else t


def attend(cache, q, slot, pos, window=0, sinks=0):
    """q [heads, d] at `pos` of a slot: the output in 64 bits, and how far an
    fp32 kernel may be from it. Scores: a sum of d products of a 24-bit query
    and an exact key, each product and addition off by at most 2^-24 of the sum
    of magnitudes (d + 2 roundings with the scale's, twice that for queries
    held in 22 bits), and exp of a score's error e scales its weight by 1 + e.
    Weights: exp and its argument in base 2 add 2^-22 of (1 + |score|), the 22
    bits of a weight 2^-22. Numerator and denominator are each off by that
    share of their magnitudes, their sums of n terms by n roundings at most, of
    which a tile's partial sums bound n by 32 + visible / 32.
    Weights are held as two fp16 numbers in a unit in which the largest of a
    row is at least 2^10 (2^(score - reference + 10), and the reference is one
    of the scores). fp16's smallest step is 2^-24, so besides its 22 bits a
    weight may be off by 2^-25 / 2^10 = 2^-35 of the largest one. That matters
    where the largest weight meets a value of zero: it is 2^-35 times the sum
    of |v|, whatever the other weights. A prefill's weights also carry their
    block's value scale relative to the largest of a tile, up to a ratio of
    2^6 (beyond it blocks are summed one by one): as much more, at most.
    """
    heads, d = q.shape
    kv = cache.q["k"].shape[1]
    t = visible(pos, window, sinks)
    out, tol = np.zeros((heads, d)), np.zeros((heads, d))
    for h in range(heads):
        g = h // (heads // kv)
        k, v = cache.value("k", slot, g, t), cache.value("v", slot, g, t)
        x = q[h].astype(np.float64)
        s = k @ x / np.sqrt(d)
        size = np.abs(k) @ np.abs(x) / np.sqrt(d)
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ v
        share = 2 * (d + 2) * 2.0 ** -24 * size.max() + 2.0 ** -22 * (2 + 2 * np.abs(s).max())
        share += (34 + len(t) / 32) * 2.0 ** -24
        used = cache.s["v"][slot, g, np.unique(t // cache.block)]
        spread = min(64.0, used.max() / used[used > 0].min()) if (used > 0).any() else 1.0
        tol[h] = 2 * share * (p @ np.abs(v)) + 2 * 2.0 ** -35 * spread * p.max() * np.abs(v).sum(0) + 1e-30
    return out, tol
