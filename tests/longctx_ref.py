"""The long-context serving operators in 64 bits, from their definitions in
include/i4d.h, token by token (numpy on the host)."""
import math

import numpy as np

TOP = {"int8": 127.0, "e4m3": 448.0}


def frequencies(rot, base=10000.0, scaling="none", factor=1.0, original=4096, low=1.0, high=32.0):
    if scaling == "base":
        base = base * factor ** (rot / (rot - 2.0))
    f = np.array([base ** (-2.0 * i / rot) for i in range(rot // 2)])
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        g = np.clip((original * f / (2 * math.pi) - low) / (high - low), 0.0, 1.0)
        f = f * (g + (1 - g) / factor)
    return f


def rope(x, positions, freq, magnitude, interleaved, inverse=False):
    """x [tokens, heads, dim] float64."""
    y = x.copy()
    half = len(freq)
    for t, p in enumerate(positions):
        ang = (-1.0 if inverse else 1.0) * float(p) * freq
        c, s = np.cos(ang) * magnitude, np.sin(ang) * magnitude
        a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
        u, v = x[t][:, a], x[t][:, b]
        y[t][:, a], y[t][:, b] = u * c - v * s, v * c + u * s
    return y


def power_scale(top, kind):
    """Least power of two s >= 2^-126 with top <= TOP * s."""
    e = -126
    while top > TOP[kind] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def nearest(y, kind):
    """Nearest code values of y (float64), ties to even; NaN 0, beyond the range the largest."""
    y = np.clip(np.where(np.isnan(y), 0.0, y), -TOP[kind], TOP[kind])
    if kind == "int8":
        return np.round(y)
    mag = np.abs(y)
    step = 2.0 ** (np.floor(np.log2(np.maximum(mag, 2.0 ** -6))) - 3)
    return np.round(y / step) * step


class Cache:
    """Code values [blocks, heads, block_tokens, dim] and scales, as float64."""

    def __init__(self, k, v, k_scale, v_scale, kind):
        self.codes = [np.array(k, np.float64), np.array(v, np.float64)]
        self.scale = [np.array(k_scale, np.float64), np.array(v_scale, np.float64)]
        self.kind = kind
        self.bs = k.shape[2]

    def append(self, new, q_start, lengths, table):
        """new: (k, v) [tokens, heads, dim] float64."""
        for which in range(2):
            codes, scale = self.codes[which], self.scale[which]
            for b, length in enumerate(lengths):
                x = new[which][q_start[b]:q_start[b + 1]]
                first = length - len(x)
                for j in range(first // self.bs, -(-length // self.bs)):
                    lo, hi, blk = max(first, j * self.bs), min(length, (j + 1) * self.bs), table[b][j]
                    if not 0 <= blk < len(codes) or lo >= hi:
                        continue
                    part = x[lo - first:hi - first]
                    for h in range(codes.shape[1]):
                        y = part[:, h]
                        fin = np.abs(y[np.isfinite(y)])
                        s = power_scale(fin.max() if fin.size else 0.0, self.kind)
                        old = lo - j * self.bs
                        if old:
                            s = max(s, scale[blk, h])
                            codes[blk, h, :old] = nearest(codes[blk, h, :old] * (scale[blk, h] / s), self.kind)
                        scale[blk, h] = s
                        codes[blk, h, old:hi - j * self.bs] = nearest(y / s, self.kind)

    def tokens(self, which, table_row, head, idx):
        """Values of one head's tokens at cache indices idx."""
        blk = np.asarray(table_row)[np.asarray(idx) // self.bs]
        return self.codes[which][blk, head, np.asarray(idx) % self.bs] * self.scale[which][blk, head][:, None]

    def evict(self, table, lengths, weights, budget, recent):
        """In place: (lengths, kept indices [b][h], weights); weights keep zeros up to the old length."""
        out_w, keep, lens = weights.copy(), [], []
        for b, length in enumerate(lengths):
            lens.append(min(length, budget))
            rows = []
            for h in range(self.codes[0].shape[1]):
                if length <= budget:
                    rows.append(np.arange(length))
                    continue
                w = weights[b, h, :length - recent]
                order = sorted(range(len(w)), key=lambda i: (-w[i] if w[i] == w[i] else math.inf, i))
                at = np.array(sorted(order[:budget - recent]) + list(range(length - recent, length)), dtype=np.int64)
                rows.append(at)
                out_w[b, h, :length] = 0
                out_w[b, h, :budget] = weights[b, h][at]
                row = np.asarray(table[b])
                for which in range(2):
                    codes, scale = self.codes[which], self.scale[which]
                    moved, had = codes[row[at // self.bs], h, at % self.bs], scale[row[at // self.bs], h]
                    for j in range(-(-budget // self.bs)):
                        part = slice(j * self.bs, min(budget, (j + 1) * self.bs))
                        top = had[part].max()
                        ratio = had[part] / top if top > 0 else had[part] * 0
                        codes[row[j], h, :part.stop - part.start] = nearest(moved[part] * ratio[:, None], self.kind)
                        scale[row[j], h] = top
            keep.append(rows)
        return lens, keep, out_w


def attention(cache, q, q_start, lengths, table, scale, window=0):
    """out, lse [tokens, heads], probabilities' sums [batch][heads][length], and for
    error bounds sum p |v| (like out) and the largest sum |q k| scale of a row (like lse)."""
    heads, dim = q.shape[1:]
    kv = cache.codes[0].shape[1]
    group = heads // kv
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    lse, size = np.full(q.shape[:2], -np.inf), np.zeros(q.shape[:2])
    sums = []
    for b, length in enumerate(lengths):
        n = q_start[b + 1] - q_start[b]
        sums.append(np.zeros((kv, length)))
        good = np.array([0 <= table[b][j // cache.bs] < len(cache.codes[0]) for j in range(length)], bool)
        idx = np.arange(length)[good]
        if not n or not len(idx):
            continue
        for h in range(kv):
            k, v = cache.tokens(0, table[b], h, idx), cache.tokens(1, table[b], h, idx)
            for a in range(h * group, (h + 1) * group):
                for i in range(n):
                    pos, row = length - n + i, q_start[b] + i
                    see = idx <= pos
                    if window:
                        see &= idx > pos - window
                    if not see.any():
                        continue
                    x = q[row, a]
                    s = (k[see] @ x) * scale
                    size[row, a] = np.max(np.abs(k[see]) @ np.abs(x)) * abs(scale)
                    m = s.max()
                    e = np.exp(s - m)
                    lse[row, a] = m + np.log(e.sum())
                    p = e / e.sum()
                    out[row, a], mag[row, a] = p @ v[see], p @ np.abs(v[see])
                    sums[b][h, idx[see]] += p
    return out, lse, sums, mag, size


def logits(x, history, prompt_len, repetition, frequency, presence, bias, allowed):
    """One row: history (ids), bias (list of (id, value)), allowed (booleans); None where absent."""
    y = x.copy()
    v = len(x)
    hist = [i for i in history if 0 <= i < v] if history is not None else []
    late = [i for n, i in enumerate(history) if n >= prompt_len and 0 <= i < v] if history is not None else []
    for i in set(hist):
        if repetition is not None:
            y[i] = y[i] / repetition if y[i] > 0 else y[i] * repetition
        n = late.count(i)
        if n:
            y[i] -= (frequency or 0.0) * n + (presence or 0.0)
    for i, b in bias or []:
        if 0 <= i < v:
            y[i] += b
    if allowed is not None:
        y[~allowed] = -np.inf
    return y
