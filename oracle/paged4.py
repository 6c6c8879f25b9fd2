"""The paged 4-bit KV cache in float64 numpy, from its definition: the tables and
the attention are oracle.paged's, the codes are its own.  Nothing here is taken
from the product's code.

A head's 128 values are four groups of 32.  A group's scale is its largest
magnitude over 7, rounded to 8 significant bits, in multiples of 2^-24 and from
2^-24 to 9344 (0 without a value but 0), its codes are the values over it,
rounded to the nearest whole number (ties to even), at most 7 in magnitude.  A group with
a value that is not finite stands for NaN.
"""
import numpy as np

from .paged import D, PAGE, Cache, pages_of

GROUP = 32


def code(x):
    """(codes (..., 4, 32), scales (..., 4)) of x (..., 128) float64."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], D // GROUP, GROUP)
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    top = np.abs(g).max(-1)
    y = top / 7                                    # off by 2^-53: no tie of 8 bits is that near to another number
    step = 2.0 ** np.maximum(np.frexp(y)[1] - 8.0, -24.0)
    s = np.clip(np.rint(y / step) * step, 2.0 ** -24, 9344.0)
    n = np.clip(np.rint(g / s[..., None]), -7, 7)
    s = np.where(bad, np.nan, np.where(top > 0, s, 0.0))
    return np.where((top > 0)[..., None], n, 0.0), s


class Cache4(Cache):
    def __init__(self, n_seqs, max_len, n_pages, n_kv):
        super().__init__(n_seqs, max_len, n_pages, n_kv)
        self.exps = None
        self.scales = [np.zeros((n_pages, n_kv, PAGE, D // GROUP)) for _ in "kv"]

    def append(self, k, v, plan):
        for t, slot in enumerate(plan["slots"][:len(k)]):
            if slot < 0:
                continue
            for x, codes, scales in ((k, self.codes[0], self.scales[0]), (v, self.codes[1], self.scales[1])):
                n, s = code(x[t])
                codes[slot // PAGE, :, slot % PAGE] = n.reshape(self.n_kv, D)
                scales[slot // PAGE, :, slot % PAGE] = s

    def held(self, row, n):
        ids = self.table[row, :pages_of(n)]
        return [np.concatenate([c[p] * np.repeat(s[p], GROUP, -1) for p in ids], 1)[:, :n] if n else np.zeros((self.n_kv, 0, D))
                for c, s in zip(self.codes, self.scales)]

    def fetch(self, first, count):
        """(k, v, cu): the rows' positions one behind the other."""
        cu, parts = [0], ([], [])
        for i, c in enumerate(count):
            f = min(max(first[i], 0), self.lens[i])
            c = min(max(c, 0), self.lens[i] - f)
            cu.append(cu[-1] + c)
            for x, to in zip(self.held(i, f + c), parts):
                to.append(x[:, f:f + c].transpose(1, 0, 2))
        return [np.concatenate(x) for x in parts] + [cu]

    def attend(self, q, plan, scale):
        """(out, bound): oracle.paged's, and what the cut of small weights adds.
        Weights enter the products times 2^6 at least of a wave's largest, with
        2^-24 as the last place: 2^-30 of sum |v| over what a row sees."""
        out, bound = super().attend(q, plan, scale)
        group = q.shape[1] // self.n_kv
        for i in range(self.n_seqs):
            now, past, t0 = plan["kv_len"][i], plan["past"][i], plan["cu"][i]
            n = plan["cu"][i + 1] - t0
            if now == 0 or n == 0:
                continue
            v = np.nan_to_num(np.abs(self.held(i, now)[1]))
            sums = np.cumsum(v, 1)[:, past:past + n]            # (heads, n, 128)
            bound[t0:t0 + n] += 2.0 ** -30 * np.repeat(sums.transpose(1, 0, 2), group, 1)
        return out, bound
