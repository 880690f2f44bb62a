"""Plain 64-bit forms of the operators on a decoder's int8 cache and of verify_drafts, and how far a result may lie from them.

A rounding is off by at most half a step, relative to the value: 2**-24 in fp32 (U below), 2**-11 in fp16, 2**-8 in bf16."""
import numpy as np

U = 2.0 ** -24
HALF_STEP = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


class Cache:
    """Codes [pages, heads, page, dim] and scales [pages, heads] of keys and values."""

    def __init__(self, pages, heads, page, dim, rng=None):
        shape = (pages, heads, page, dim)
        if rng is None:
            rng = np.random.default_rng(pages * 1000 + dim)
        self.codes = [np.clip(np.rint(rng.standard_normal(shape) * 35), -127, 127).astype(np.int8) for _ in range(2)]
        self.scales = [(rng.uniform(0.6, 1.4, (pages, heads)) / 35).astype(np.float32) for _ in range(2)]
        self.pages, self.heads, self.page, self.dim = shape

    def copy(self):
        c = object.__new__(Cache)
        c.codes, c.scales = [x.copy() for x in self.codes], [x.copy() for x in self.scales]
        c.pages, c.heads, c.page, c.dim = self.pages, self.heads, self.page, self.dim
        return c


def sequences(rows, seqs, width, page, lengths, offsets):
    """(first row, new tokens, position of the first) of each sequence."""
    o = np.arange(seqs + 1) * (rows // seqs) if offsets is None else np.clip(np.asarray(offsets, np.int64), 0, rows)
    n = np.clip(np.asarray(lengths, np.int64), 0, width * page)
    return [(int(o[s]), int(max(0, o[s + 1] - o[s])), int(n[s] - max(0, o[s + 1] - o[s]))) for s in range(seqs)]


def page_of(cache, table, s, pos):
    at = pos // cache.page
    if pos < 0 or at >= table.shape[1]:
        return -1
    p = int(table[s, at])
    return p if 0 <= p < cache.pages else -1


def write(cache, new, table, lengths, offsets):
    """Changes `cache`; new: (k, v) float64 [rows, heads, dim]."""
    seqs, width = table.shape
    for kv in range(2):
        codes, scales, x = cache.codes[kv], cache.scales[kv], new[kv]
        for s, (row, n, first) in enumerate(sequences(len(x), seqs, width, cache.page, lengths, offsets)):
            for start in range(max(first, 0) // cache.page * cache.page, first + n, cache.page):
                lo, hi = max(start, first, 0), min(start + cache.page, first + n)
                p = page_of(cache, table, s, start)
                if p < 0 or hi <= lo:
                    continue
                for h in range(cache.heads):
                    mine = x[row + lo - first:row + hi - first, h]
                    old = np.float32(0) if lo == start else scales[p, h]
                    with np.errstate(all="ignore"):
                        scale = max(old, np.float32(np.abs(mine).max() / 127)) if np.isfinite(mine).all() and old == old else np.float32(np.nan)
                        if not np.isfinite(scale):
                            codes[p, h, lo - start:hi - start] = 0
                        elif scale == 0:
                            codes[p, h, lo - start:hi - start] = 0
                        else:
                            codes[p, h, lo - start:hi - start] = np.clip(np.rint(mine / np.float64(scale)), -127, 127)
                            if scale > old:
                                c = codes[p, h, :lo - start].astype(np.float64)
                                codes[p, h, :lo - start] = np.clip(np.rint(c * np.float64(old) / np.float64(scale)), -127, 127)
                    scales[p, h] = scale


def read(cache, kv, rows, table, lengths, offsets):
    """float64 [rows, heads, dim] and which rows belong to a sequence."""
    out, there = np.zeros((rows, cache.heads, cache.dim)), np.zeros(rows, bool)
    seqs, width = table.shape
    for s, (row, n, first) in enumerate(sequences(rows, seqs, width, cache.page, lengths, offsets)):
        for i in range(n):
            there[row + i] = True
            p = page_of(cache, table, s, first + i)
            if p >= 0:
                out[row + i] = cache.codes[kv][p, :, (first + i) % cache.page].astype(np.float64) * cache.scales[kv][p].astype(np.float64)[:, None]
    return out, there


def attention(cache, q, table, lengths, offsets, kind, scale=None, window=0, sinks=0):
    """(out, how far off it may be, lse, how far off it may be, rows of sequences) of q float64 [rows, heads, dim].

    A score x is a sum of dim products of exact codes with q, which is exact or (few rows) rounded to whole numbers of which the row's largest is 2^19 (2^26 for f32) at least,
    half a step of which is 2^-20 (2^-27) of that value; added exactly or in fp32 with at most one step (2 U) of the sum of magnitudes for each, times three factors: off by
    dx = 2 U (dim + 2) scale sum |q k| + 2^-20 scale max |q| sum |k| and, with the difference to the maximum and the power of two, by 6 U |x - max| + 8 U relative to the weight.  A weight in f16 is
    off by 2**-11, in two f16 numbers by 2**-22, and by 2**-31 of the largest weight times the largest value where it is tiny
    (the rounding below f16's least numbers, of weights that are at least 2**6 at the largest).  Sums over n tokens are
    added in fp32, 16 at a time, and rescaled at most every 32: n / 4 + 64 steps in all."""
    rows, heads, dim = q.shape
    group = heads // cache.heads
    scale = dim ** -0.5 if scale is None else scale
    out, off, lse, lse_off, there = np.zeros(q.shape), np.zeros(q.shape), np.full((rows, heads), -np.inf), np.zeros((rows, heads)), np.zeros(rows, bool)
    seqs, width = table.shape
    h16 = 2.0 ** -22 if kind == "f32" else 2.0 ** -11
    for s, (row, n, first) in enumerate(sequences(rows, seqs, width, cache.page, lengths, offsets)):
        length = first + n
        pos = np.arange(max(length, 0))
        pages = np.array([page_of(cache, table, s, p) for p in range(0, max(length, 0), cache.page)] or [-1])
        where, slot = pages[pos // cache.page], pos % cache.page
        known = where >= 0
        for h in range(cache.heads):
            w0 = np.where(known, where, 0)
            k = cache.codes[0][w0, h, slot].astype(np.float64) * cache.scales[0][w0, h].astype(np.float64)[:, None]
            v = cache.codes[1][w0, h, slot].astype(np.float64) * cache.scales[1][w0, h].astype(np.float64)[:, None]
            for i in range(n):
                there[row + i] = True
                at = first + i
                seen = known & (pos <= at)
                if window > 0:
                    seen &= (pos > at - window) | (pos < sinks)
                if not seen.any():
                    continue
                j = np.flatnonzero(seen)
                for g in range(h * group, (h + 1) * group):
                    with np.errstate(all="ignore"):
                        x = (k[j] @ q[row + i, g]) * scale
                        size = (np.abs(k[j]) @ np.abs(q[row + i, g])) * abs(scale)
                        top = x.max()
                        e = np.exp(x - top)
                        w = e / e.sum()
                        out[row + i, g] = w @ v[j]
                        dx = (2 * U * (dim + 2) * size + (2.0 ** -27 if kind == "f32" else 2.0 ** -20) * abs(scale) * np.abs(q[row + i, g]).max() * np.abs(k[j]).sum(1)).max()
                        dw = 2 * (dx + 8 * U + 6 * U * np.abs(x - top))
                        mean = w @ np.abs(v[j])
                        wide = 2 * U * (len(j) / 4 + 64)
                        o = (w * (dw + h16)) @ np.abs(v[j]) + mean * (w @ dw + 2 * wide) + 2.0 ** -31 * w.max() * np.abs(v[j]).max() * len(j)
                        off[row + i, g] = o + HALF_STEP[kind] * (np.abs(out[row + i, g]) + o) + LEAST[kind]
                        lse[row + i, g] = top + np.log(e.sum())
                        lse_off[row + i, g] = (w @ dw) + wide + 8 * U * (1 + abs(lse[row + i, g]) + abs(top))
    return out, off, lse, lse_off, there


def verify(target, drafted, tokens, accept, sample, offsets):
    """(accepted, next) of float64 probabilities."""
    seqs, drafts, vocab = len(sample), len(tokens), target.shape[1]
    o = np.arange(seqs + 1) * (drafts // seqs) if offsets is None else offsets
    accepted, following = np.zeros(seqs, np.int32), np.zeros(seqs, np.int32)
    for s in range(seqs):
        n, b, e = 0, int(o[s]), int(o[s + 1])
        while b + n < e:
            t = int(tokens[b + n])
            if t < 0:
                e = b + n
                break
            if t >= vocab or not float(accept[b + n]) * (1.0 if drafted is None else drafted[b + n, t]) < target[b + n + s, t]:
                break
            n += 1
        r = target[b + n + s].copy()
        if b + n < e:
            if drafted is not None:
                r = r - drafted[b + n]
            elif tokens[b + n] < vocab:
                r[tokens[b + n]] -= 1.0
        clean = lambda r: np.where((r > 0) & np.isfinite(r), r, 0.0)  # noqa: E731
        r = clean(r)
        if r.sum() == 0:
            r = clean(target[b + n + s])
        accepted[s] = n
        if r.sum() == 0:
            following[s] = -1
            continue
        sums = np.cumsum(r)
        above = np.flatnonzero((sums > float(sample[s]) * sums[-1]) & (r > 0))
        following[s] = above[0] if len(above) else np.flatnonzero(r > 0)[-1]
    return accepted, following
