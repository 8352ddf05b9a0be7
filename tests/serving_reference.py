"""What the steps between the linears compute, in numpy's 64 bits and written from their definitions: the plan of pages and
slots, the paged 8-bit cache, attention over it, and the choice of the next token."""
import numpy as np


def plan(past, fresh, table, free, page, rows, taken=0):
    """(table, lens, starts, slots, positions, taken)"""
    table, starts = table.copy(), [0]
    slots, positions = np.full(rows, -1, np.int64), np.zeros(rows, np.int32)
    for i, (p, f) in enumerate(zip(past, fresh)):
        p, f = max(int(p), 0), max(int(f), 0)
        for col in range(-(-p // page), -(-(p + f) // page)):
            if col < table.shape[1]:
                table[i, col] = free[taken] if taken < len(free) else -1
            taken += 1
        for j in range(f):
            row, at = starts[-1] + j, p + j
            if row < rows:
                entry = int(table[i, at // page]) if at // page < table.shape[1] else -1
                slots[row] = entry * page + at % page if entry >= 0 else -1
                positions[row] = at
        starts.append(starts[-1] + f)
    lens = np.array([max(int(p), 0) + max(int(f), 0) for p, f in zip(past, fresh)], np.int32)
    return table, lens, np.array(starts, np.int32), slots, positions, taken


def away(x):
    return np.sign(x) * np.floor(np.abs(x) + 0.5)


class Cache:
    """Codes [pages, heads, page, dim] of either side and their scales."""

    def __init__(self, pages, heads, page, dim):
        self.page = page
        self.codes = {s: np.zeros((pages, heads, page, dim), np.int64) for s in "kv"}
        self.scales = {s: np.zeros((pages, heads), np.float32) for s in "kv"}

    def write(self, k, v, slots):
        for side, x in (("k", k), ("v", v)):
            x = np.asarray(x, np.float64)
            for p in np.unique(slots[slots >= 0] // self.page):
                if p >= len(self.scales["k"]):
                    continue
                mine = np.flatnonzero((slots >= 0) & (slots // self.page == p))
                places = slots[mine] % self.page
                old = np.float32(0) if (places == 0).any() else self.scales[side][p]
                new = x[mine]
                finite = np.where(np.isfinite(new), np.abs(new), 0.0).max((0, 2))
                scale = np.maximum(old, finite.astype(np.float32) / np.float32(127)).astype(np.float32)
                scale[scale < np.float32(2.0 ** -126)] = 0
                s = np.where(scale > 0, scale, 1).astype(np.float64)[:, None, None]
                codes = away(self.codes[side][p] * np.broadcast_to(np.asarray(old, np.float64), scale.shape)[:, None, None] / s)
                with np.errstate(invalid="ignore"):
                    for i, place in enumerate(places):
                        q = np.clip(away(new[i] / s[:, 0]), -127, 127)
                        codes[:, place] = np.where(np.isnan(new[i]), 0, q)
                codes[scale == 0] = 0
                self.codes[side][p] = codes.astype(np.int64)
                self.scales[side][p] = scale

    def values(self, side, page):
        """[heads, page, dim]"""
        return self.codes[side][page] * self.scales[side][page].astype(np.float64)[:, None, None]


def attention(q, cache, table, lens, starts, scale, window, out):
    """Rows of `out` that belong to a sequence, replaced; also the most that the scores of a row can be off for a relative error
    of one in its largest query value (what an 8-bit or 16-bit split of q costs goes by it), and the largest |v|."""
    out = np.array(out, np.float64)
    reach, most = np.zeros(out.shape[:2]), np.zeros(out.shape[:2])
    heads, dim = q.shape[1:]
    page, pages, group = cache.page, len(cache.scales["k"]), heads // cache.codes["k"].shape[1]
    for i, length in enumerate(lens):
        length = int(length)
        entries = [int(e) for e in table[i][:-(-max(length, 0) // page)]]
        at = np.concatenate([np.arange(c * page, min((c + 1) * page, length)) for c, e in enumerate(entries) if 0 <= e < pages] or [np.arange(0)])
        have = [e for e in entries if 0 <= e < pages]
        if have and at.size:
            k = np.concatenate([cache.values("k", e) for e in have], 1)
            v = np.concatenate([cache.values("v", e) for e in have], 1)
            full = np.concatenate([np.arange(c * page, (c + 1) * page) for c, e in enumerate(entries) if 0 <= e < pages])
            k, v = k[:, full < length], v[:, full < length]
        for r in range(int(starts[i]), min(int(starts[i + 1]), len(q))):
            pos = length - int(starts[i + 1]) + r
            seen = (at <= pos) & ((at > pos - window) if window else True)
            for h in range(heads):
                if not seen.any():
                    out[r, h] = 0
                    continue
                kk, vv, x = k[h // group][seen], v[h // group][seen], q[r, h].astype(np.float64)
                s = kk @ x * scale
                p = np.exp(s - s.max())
                out[r, h] = (p / p.sum()) @ vv
                reach[r, h] = scale * np.abs(kk).sum(1).max() * np.abs(x).max()
                most[r, h] = np.abs(vv).max()
    return out, reach, most


def sample(logits, uniform, temperature, top_k=None, top_p=None, min_p=None):
    """(tokens, probabilities)"""
    tokens, probs = [], []
    for r, row in enumerate(np.asarray(logits, np.float64)):
        order = np.argsort(-np.where(np.isnan(row), -np.inf, row), kind="stable")
        order = order[row[order] > -np.inf]
        if not order.size:
            tokens.append(-1)
            probs.append(0.0)
            continue
        t = float(temperature[r])
        if not t > 0:
            tokens.append(int(order[0]))
            probs.append(1.0)
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            x = (row[order] - row[order[0]]) / t
        w = np.exp(np.where(row[order] == row[order[0]], 0.0, x))
        kept = w[:int(top_k[r])] if top_k is not None and top_k[r] > 0 else w
        if top_p is not None and top_p[r] < 1:
            sums = np.cumsum(kept)
            kept = kept[:int((sums < float(top_p[r]) * sums[-1]).sum()) + 1]
        if min_p is not None:
            kept = kept[:max(1, int((w >= float(min_p[r])).sum()))]
        sums = np.cumsum(kept)
        i = min(int((sums <= float(uniform[r]) * sums[-1]).sum()), len(kept) - 1)
        tokens.append(int(order[i]))
        probs.append(kept[i] / sums[-1])
    return np.array(tokens), np.array(probs)
