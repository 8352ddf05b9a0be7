"""What the head norms, the rotation, the 4-bit cache, attention over it and the check of drafted tokens compute, in numpy's 64 bits and
written from their definitions."""
import math

import numpy as np

LADDER = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def rope(x, positions, frequencies, axis=None, weight=None, eps=1e-6, neighbours=False, factor=1.0):
    """Heads [rows, heads, dim], normed and rotated; positions [rows] or [axes, rows]."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * np.asarray(weight, np.float64)
    y, positions = x.copy(), np.atleast_2d(positions)
    n = len(frequencies)
    for i, f in enumerate(np.asarray(frequencies, np.float64)):
        pos = positions[min(int(axis[i]), len(positions) - 1) if axis is not None else 0]
        angle = (pos.astype(np.float64) * f)[:, None]
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + n)
        c, s = np.cos(angle) * np.float64(np.float32(factor)), np.sin(angle) * np.float64(np.float32(factor))
        y[:, :, a], y[:, :, b] = x[:, :, a] * c - x[:, :, b] * s, x[:, :, a] * s + x[:, :, b] * c
    return y


def quantize(x):
    """Blocks of 32 along the last axis: codes (uint8, one each) and powers (uint8)."""
    x = np.asarray(x, np.float64)
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    finite = np.where(np.abs(blocks) <= np.finfo(np.float32).max, np.abs(blocks), 0.0)
    most = finite.max(-1)
    power = np.full(most.shape, -96)
    for e in range(-96, 125):
        power = np.where(most >= 7 * 2.0 ** e, e + 1, power)
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.abs(blocks) / 2.0 ** power[..., None]
        border = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
        code = np.zeros(blocks.shape, np.int64)
        for i, b in enumerate(border):       # between codes i and i + 1; a half goes to the even one
            code += (y > b) if i % 2 == 0 else (y >= b)
        code += 8 * (blocks < 0)
    return code.reshape(x.shape).astype(np.uint8), (power + 127).astype(np.uint8)


def values(codes, powers):
    codes = np.asarray(codes)
    mag = LADDER[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    p = np.where(powers == 255, np.nan, 2.0 ** (powers.astype(np.float64) - 127))
    return (mag.reshape(*codes.shape[:-1], -1, 32) * p[..., None]).reshape(codes.shape)


class Cache:
    """Codes [pages, heads, page, dim], one to a byte, and powers [pages, heads, page, dim / 32] of either side."""

    def __init__(self, pages, heads, page, dim, seed=None, powers=(124, 128)):
        self.page, self.dim = page, dim
        g = np.random.default_rng(seed)
        make = (lambda lo, hi, *s: np.zeros(s, np.uint8)) if seed is None else (lambda lo, hi, *s: g.integers(lo, hi, s).astype(np.uint8))
        self.codes = {s: make(0, 16, pages, heads, page, dim) for s in "kv"}
        self.powers = {s: make(*powers, pages, heads, page, dim // 32) for s in "kv"}

    def write(self, k, v, slots):
        for side, x in (("k", k), ("v", v)):
            codes, powers = quantize(x)
            for i, s in enumerate(np.asarray(slots)):
                if 0 <= s < self.page * len(self.codes["k"]):
                    self.codes[side][s // self.page, :, s % self.page] = codes[i]
                    self.powers[side][s // self.page, :, s % self.page] = powers[i]

    def values(self, side, page):
        """[heads, page, dim]"""
        return values(self.codes[side][page], self.powers[side][page])

    def tensors(self):
        """k, v, k_powers, v_powers as the cache has them."""
        pages, heads, page, dim = self.codes["k"].shape
        pair = lambda c: c[..., 0::2] | c[..., 1::2] << 4  # noqa: E731
        v = pair(self.codes["v"]).reshape(pages, heads, page // 4, 4, 16, dim // 32).swapaxes(3, 4)
        return tuple(np.ascontiguousarray(t) for t in (pair(self.codes["k"]), v, self.powers["k"], self.powers["v"].swapaxes(2, 3)))


def attention(q, cache, table, lens, starts, scale, window, cap, out):
    """Rows of `out` that belong to a sequence, replaced; per row and head also the largest sum of |q k| scale of a score, and the largest |v|."""
    out = np.array(out, np.float64)
    reach, most = np.zeros(out.shape[:2]), np.zeros(out.shape[:2])
    heads = q.shape[1]
    page, pages, group = cache.page, len(cache.codes["k"]), heads // cache.codes["k"].shape[1]
    for i, length in enumerate(int(n) for n in lens):
        have = [(c, int(e)) for c, e in enumerate(table[i][:-(-max(length, 0) // page)]) if 0 <= e < pages]
        at = np.concatenate([np.arange(c * page, (c + 1) * page) for c, _ in have] or [np.arange(0)])
        if have:
            k, v = (np.concatenate([cache.values(s, e) for _, e in have], 1)[:, at < length] for s in "kv")
            at = at[at < length]
        for r in range(int(starts[i]), min(int(starts[i + 1]), len(q))):
            pos = length - int(starts[i + 1]) + r
            seen = (at <= pos) & ((at > pos - window) if window else True)
            if not seen.any():
                out[r] = 0
                continue
            for kv in range(heads // group):
                hs = slice(kv * group, (kv + 1) * group)
                kk, vv, x = k[kv][seen], v[kv][seen], q[r, hs].astype(np.float64)
                s = x @ kk.T * scale
                s = cap * np.tanh(s / cap) if cap else s
                p = np.exp(s - s.max(-1, keepdims=True))
                out[r, hs] = p / p.sum(-1, keepdims=True) @ vv
                reach[r, hs] = (np.abs(x) @ np.abs(kk).T).max(-1) * scale
                most[r, hs] = np.abs(vv).max()
    return out, reach, most


def target(row, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """The distribution that a row of logits is sampled from, by word."""
    x = np.asarray(row, np.float64)
    order = np.argsort(-np.where(np.isnan(x), -np.inf, x), kind="stable")
    order = order[x[order] > -np.inf]
    p = np.zeros(len(x))
    if not order.size:
        return p
    if not temperature > 0:
        p[order[0]] = 1
        return p
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp(np.where(x[order] == x[order[0]], 0.0, (x[order] - x[order[0]]) / temperature))
    kept = w[:top_k] if top_k > 0 else w
    if top_p < 1:
        sums = np.cumsum(kept)
        kept = kept[:int((sums < top_p * sums[-1]).sum()) + 1]
    kept = kept[:max(1, int((w >= min_p).sum()))]
    p[order[:len(kept)]] = kept / math.fsum(kept)
    return p


def verify(logits, drafted, starts, uniform, draw, temperature, top_k=None, top_p=None, min_p=None, draft=None):
    """(tokens [rows], accepted [sequences], probabilities [rows])"""
    rows = len(logits)
    tokens, probs, accepted = np.full(rows, -1), np.zeros(rows), []
    rule = lambda a, r, none: none if a is None else a[r]  # noqa: E731
    for i in range(len(starts) - 1):
        a, b, here = int(starts[i]), int(starts[i + 1]), 0
        for r in range(a, b):
            p = target(logits[r], float(temperature[r]), int(rule(top_k, r, 0)), float(rule(top_p, r, 1.0)), float(rule(min_p, r, 0.0)))
            if not p.any():
                break
            left = p
            if r < b - 1:
                word = int(drafted[r])
                inside = 0 <= word < len(p)
                q = (1.0 if draft is None else float(draft[r][word])) if inside else 0.0
                if inside and float(uniform[r]) * q < p[word]:
                    tokens[r], probs[r] = word, p[word]
                    here += 1
                    continue
                if draft is None:
                    left = p.copy()
                    left[word if inside else slice(0, 0)] = 0
                else:
                    left = np.maximum(p - np.asarray(draft[r], np.float64), 0)
                left = left if left.sum() > 0 else p
            sums = np.cumsum(left)
            word = min(int((sums <= float(draw[i]) * sums[-1]).sum()), int((sums < sums[-1]).sum()))
            tokens[r], probs[r] = word, p[word]
            break
        accepted.append(here)
    return tokens, np.array(accepted), probs
