"""The paged 8-bit KV cache, its rotary positions and its attention in float64
numpy and plain Python, from their definitions.  Nothing here is taken from the
product's code.

A cache holds rows (sequences) in pages of 64 positions.  Per page and kv head
the values of k, and those of v, are e4m3 codes times 2^e, e the smallest
integer in [-40, 60] for which 448 2^e reaches the largest finite value the
page has been given (-40 without one).  Values that are not finite, or past
448 2^60, are NaN.
"""
import math
from fractions import Fraction

import numpy as np

PAGE = 64
D = 128
E_MIN, E_MAX = -40, 60
TWO_PI = Fraction("6.2831853071795864769252867665590057683943387987502")


def pages_of(n):
    return -(-n // PAGE)


def code(x, e):
    """e4m3 nearest to x / 2^e, ties to even, as float64; NaN past 448."""
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.asarray(x, np.float64) / 2.0 ** e
        mag = np.where(np.isfinite(y), np.abs(y), 1.0)
        step = 2.0 ** (np.frexp(np.maximum(mag, 2.0 ** -6))[1] - 1 - 3)
        r = np.where(np.abs(y) <= 448.0, np.rint(y / step) * step, np.nan)
    return r


def exponent(x):
    """e of the values x: see above."""
    a = np.abs(np.asarray(x, np.float64))
    a = a[np.isfinite(a)]
    top = float(a.max()) if a.size else 0.0
    if top == 0.0:
        return E_MIN
    m, b = math.frexp(top)                       # top = m 2^b, 1/2 <= m < 1; 448 = 7/8 2^9
    return min(max(b - 9 + (m > 0.875), E_MIN), E_MAX)


def rotate(x, positions, freqs, magnitude, layout):
    """x (tokens, heads, dim) float64 turned by positions * freqs radians, the
    angle reduced exactly."""
    y = np.array(x, np.float64)
    rot = 2 * len(freqs)
    for t, p in enumerate(positions):
        for j, f in enumerate(freqs):
            a, b = (j, j + rot // 2) if layout == "half" else (2 * j, 2 * j + 1)
            ang = float(int(p) * Fraction(f) % TWO_PI)
            c, s = magnitude * math.cos(ang), magnitude * math.sin(ang)
            u, v = x[t, :, a], x[t, :, b]
            y[t, :, a], y[t, :, b] = u * c - v * s, u * s + v * c
    return y


class Cache:
    def __init__(self, n_seqs, max_len, n_pages, n_kv):
        self.n_seqs, self.max_len, self.n_kv = n_seqs, max_len, n_kv
        self.width = pages_of(max_len)
        self.table = -np.ones((n_seqs, self.width), np.int64)
        self.lens = [0] * n_seqs
        self.free = list(range(n_pages))[::-1]
        self.codes = [np.zeros((n_pages, n_kv, PAGE, D)) for _ in "kv"]
        self.exps = [np.full((n_pages, n_kv), E_MIN) for _ in "kv"]

    def extend(self, new, max_tokens, max_new):
        """The plan: dict of cu, positions, slots, kv_len, rejected, past."""
        cu, past = [0], list(self.lens)
        for n in new:
            cu.append(cu[-1] + max(n, 0))
        pos, slots = -np.ones(max_tokens, np.int64), -np.ones(max_tokens, np.int64)
        kv, rejected, wanted, pool = [], [], 0, len(self.free)
        for i, n in enumerate(new):
            n = max(n, 0)
            old, now = self.lens[i], self.lens[i] + n
            ok = now <= self.max_len and n <= max_new and cu[i + 1] <= max_tokens
            need = pages_of(now) - pages_of(old) if ok else 0
            wanted += need
            ok = ok and (need == 0 or wanted <= pool)
            rejected.append(0 if ok else 1)
            kv.append(now if ok else 0)
            if not ok:
                continue
            for j in range(pages_of(old), pages_of(now)):
                self.table[i, j] = self.free.pop()
            self.lens[i] = now
            for t in range(n):
                pos[cu[i] + t] = old + t
                slots[cu[i] + t] = self.table[i, (old + t) // PAGE] * PAGE + (old + t) % PAGE
        return {"cu": cu, "positions": pos, "slots": slots, "kv_len": kv, "rejected": rejected, "past": past}

    def rewind(self, to):
        freed = []
        for i, n in enumerate(to):
            if n < 0 or n >= self.lens[i]:
                continue
            for j in range(pages_of(n), pages_of(self.lens[i])):
                freed.append(self.table[i, j])
                self.table[i, j] = -1
            self.lens[i] = n
        self.free += freed[::-1]

    def append(self, k, v, plan):
        """k, v (tokens, n_kv, 128) of the plan's step."""
        for i in range(self.n_seqs):
            old, now = plan["past"][i], plan["kv_len"][i]
            for j in range(old // PAGE, pages_of(now) if now > old else 0):
                lo, hi = max(old, j * PAGE), min(now, (j + 1) * PAGE)
                if lo >= hi:
                    continue
                page, held = self.table[i, j], lo - j * PAGE
                rows = slice(plan["cu"][i] + lo - old, plan["cu"][i] + hi - old)
                for x, codes, exps in ((k, self.codes[0], self.exps[0]), (v, self.codes[1], self.exps[1])):
                    for h in range(self.n_kv):
                        e = exponent(x[rows, h])
                        if held:
                            e = max(e, exps[page, h])
                            codes[page, h, :held] = code(codes[page, h, :held] * 2.0 ** exps[page, h], int(e))
                        codes[page, h, held:hi - j * PAGE] = code(x[rows, h], int(e))
                        exps[page, h] = e

    def held(self, row, n):
        """(k, v) (n_kv, n, 128) that the row's first n positions stand for."""
        ids = self.table[row, :pages_of(n)]
        return [np.concatenate([c[p] * 2.0 ** e[p].astype(np.float64)[:, None, None] for p in ids], 1)[:, :n]
                for c, e in zip(self.codes, self.exps)]

    def attend(self, q, plan, scale, one_part=False):
        """(out, bound): out (tokens, n_q, 128) float64, zeros for rejected rows;
        bound is what sum p |v| and the scores' error give: per output, the
        absolute error of fp32 sums (see attend_bound).  one_part: where
        probabilities may go in one fp16 part instead of two."""
        n_q = q.shape[1]
        group = n_q // self.n_kv
        out = np.zeros((plan["cu"][-1], n_q, D))
        bound = np.zeros_like(out)
        for i in range(self.n_seqs):
            now, past, t0 = plan["kv_len"][i], plan["past"][i], plan["cu"][i]
            n = plan["cu"][i + 1] - t0
            if now == 0 or n == 0:
                continue
            k, v = self.held(i, now)
            for h in range(n_q):
                s = scale * (q[t0:t0 + n, h] @ k[h // group].T)
                mag = abs(scale) * (np.abs(q[t0:t0 + n, h]) @ np.abs(k[h // group]).T)
                hide = np.arange(now)[None, :] > past + np.arange(n)[:, None]
                s[hide] = -np.inf
                mag[hide] = 0.0
                p = np.exp(s - s.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                vv = v[h // group]
                with np.errstate(invalid="ignore"):
                    nan = np.isnan(vv)
                    y = p @ np.where(nan, 0.0, vv)
                    y[((~hide).astype(float) @ nan.astype(float)) > 0] = np.nan
                out[t0:t0 + n, h] = y
                bound[t0:t0 + n, h] = attend_bound(mag.max(1), np.abs(np.where(hide, 0, s)).max(1), now, one_part)[:, None] * (p @ np.abs(np.where(nan, 0.0, vv)))
        return out, bound


def attend_bound(mag, top, n, one_part):
    """Relative to sum p |v|: each score's fp32 sum of 128 exact products is off
    by at most 128 2^-24 mag (mag = scale sum |q k|), its product with the scale,
    the sum with v's exponent (up to 60) and the difference to the maximum by
    2^-24 of values up to 1.45 (top + 60) each; a probability is off by that and
    2^-22 of the exponential, in numerator and denominator; two fp16 parts cut
    2^-20, one part, to nearest, half a step of fp16, 2^-11 (the numerator's
    alone); sums over n positions are off by n 2^-24 each at most."""
    score = 128 * 2.0 ** -24 * mag + 4 * 2.0 ** -24 * 1.45 * (2 * top + 60)
    return 2 * (score + 2.0 ** -22 + n * 2.0 ** -24) + 2.0 ** (-11 if one_part else -20)
