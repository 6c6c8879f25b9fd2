"""Every position counts once: paged attention on values that name their
position.

Position p has the value 1 in dim p % 128 and 0 elsewhere, so an output is the
share of the weights of the positions p = dim, dim + 128, ... that its token
sees.  Weights are even, or 1, 1/2 and 1/4 in turn.  A bar is half a step of the
output's type and the bound of fp32 sums and two-part probabilities on that share
(the oracle's attend_bound, but for its sums over n terms: of an output's terms
all but n / 128 are zeros, which add without a rounding, and a sum of weights
goes by 16 of a lane and then by pages, n / 64 of them, before some dozens of
steps of lanes, waves and parts).  Every bar is checked to be less than half of
what the lightest lost or doubled position would make.
"""
import math

import pytest
import torch

import oi2
from oracle import paged as P
from tests.test_gpu_paged import dev  # noqa: F401

pytestmark = pytest.mark.gpu
D = 128

CASES = [
    # one token, up to the longest row that is not cut, and behind it
    ([0, 1, 62, 63, 64, 65], [1] * 6), ([127, 128, 255, 256, 257, 511], [1] * 6), ([959, 960, 1022, 1023, 1024, 1025], [1] * 6),
    ([1087, 1088, 2047, 2048, 5000], [1] * 5), ([20011], [1]), ([13000, 4100], [1, 1]),
    # drafts
    ([0, 61, 63, 64], [4, 4, 4, 4]), ([1021, 5003], [4, 3]), ([9000], [4]),
    # tiles of many rows and their edges
    ([0], [31]), ([0], [33]), ([0], [129]), ([0], [1300]), ([64], [257]), ([1000], [100]), ([5000], [300]), ([12345], [65]),
    # both, and rows that leave pages in the middle
    ([9000, 40, 3000, 0], [200, 1, 33, 1]), ([3, 7000, 64], [150, 1, 64]),
]


def _filled(dev, n_q, n_kv, past, new, dtype, weighted):
    c = oi2.PagedKVCache(1, n_q, n_kv, len(past), max(a + b for a, b in zip(past, new)),
                         sum(P.pages_of(a + b) for a, b in zip(past, new)) + 2, device=dev)
    c.free.copy_(torch.randperm(c.n_pages, generator=torch.Generator().manual_seed(3)).int())
    plan = None
    for lens, lo in ((past, [0] * len(past)), (new, past)):
        pos = torch.cat([torch.arange(a, a + n, device=dev) for a, n in zip(lo, lens)])
        plan = c.extend(lens, c.new_plan(max(len(pos), 1), max_new=max(max(lens), 1)))
        v = torch.zeros((len(pos), n_kv, D), device=dev, dtype=dtype)
        k = torch.zeros_like(v)
        v[torch.arange(len(pos), device=dev), :, pos % 128] = 1.0
        if weighted:
            k[:, :, 5] = -(pos % 3).to(dtype)[:, None]
        if len(pos):
            c.append(0, k, v, plan)
    return c, plan


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("past,new", CASES)
def test_every_position_counts_once(dev, dtype, past, new):
    for n_q, n_kv, weighted in ((32, 8, False), (8, 1, True), (4, 4, True)):
        print(f"[positions] {dtype} {past} + {new} heads {n_q} {n_kv} {weighted}", flush=True)
        c, plan = _filled(dev, n_q, n_kv, past, new, dtype, weighted)
        q = torch.zeros((sum(new), n_q, D), device=dev, dtype=dtype)
        ln2 = 0.0
        if weighted:
            q[:, :, 5] = math.log(2)
            ln2 = q[0, 0, 5].item()
        y = c.attend(0, q, plan, scale=1.0).double()
        t0 = 0
        for a, n in zip(past, new):
            p = torch.arange(a + n, device=dev)
            w = torch.exp(-ln2 * (p % 3).double())
            share = torch.zeros((a + n, D), dtype=torch.float64, device=dev)
            share[p, p % 128] = w
            share = share.cumsum(0)[a:]
            total = w.cumsum(0)[a:, None]
            want = share / total
            sums = ((a + n) / 128 + (a + n) / 64 + 200) * 2.0 ** -24
            tol = (torch.finfo(dtype).eps / 2 + P.attend_bound(2 * ln2, 2 * ln2, 0, False) + sums) * want
            least = math.exp(-2 * ln2) / total                     # a position's smallest share
            seen = want > 0
            # bf16 steps of long rows are coarser than a light position: those bars hold, but do not tell one
            tells = (tol < least / 2) | ~seen
            assert tells.all() or dtype == torch.bfloat16 and a + n > 4096
            err = (y[t0:t0 + n] - want[:, None]).abs()
            assert (err <= tol[:, None] + 2.0 ** -25 * (dtype == torch.float16)).all(), (a, n, float((err - tol[:, None]).max()))
            t0 += n
