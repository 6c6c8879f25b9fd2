"""What the paged attention keeps of its inputs' bits.

Every bar is half a step of the output's type and the oracle's bound for fp32
sums and two fp16 parts of a probability (attend_bound, one_part=False),
whatever the type and the number of query rows.
"""
import numpy as np
import pytest
import torch

import oi2
from oracle import paged as P
from tests.test_gpu_paged import _check_attend, _extend, _np, _pair, dev  # noqa: F401

pytestmark = pytest.mark.gpu
D = 128
DTYPES = [torch.float16, torch.bfloat16]


def _step(dev, n_q, n_kv, past, new, k, v, dtype):
    """Caches holding past positions and then the step's, of k and v (past + new
    positions a row, n_kv, 128) row after row; the plan of the step."""
    total = [a + b for a, b in zip(past, new)]
    c, o = _pair(n_kv, len(past), max(total), sum(P.pages_of(t) for t in total), dev, n_q=n_q, shuffle=1)
    at = np.cumsum([0] + total)
    for lens, lo in ((past, [0] * len(past)), (new, past)):
        plan = c.new_plan(max(sum(lens), 1), max_new=max(max(lens), 1))
        ref = _extend(c, o, plan, lens)
        rows = torch.tensor([at[i] + lo[i] + t for i, n in enumerate(lens) for t in range(n)], device=dev, dtype=torch.long)
        if len(rows):
            c.append(0, k[rows], v[rows], plan)
            o.append(_np(k[rows]), _np(v[rows]), ref)
    return c, o, plan, ref


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("past,new", [([3, 6, 1], [1, 1, 1]), ([2, 0], [2, 4]), ([0], [40]), ([0, 2], [200, 30]), ([1200], [33])])
def test_values_that_cancel(dev, dtype, past, new):
    """Nearly even weights on values 1 and -1: the result is the weights'
    difference, and shows what they were rounded to."""
    print(f"[cancel] {dtype} {past} {new}", flush=True)
    g = torch.Generator(device=dev).manual_seed(2)
    n_q, n_kv, n = 16, 4, sum(past) + sum(new)
    k = (torch.randn((n, n_kv, D), generator=g, device=dev) * 0.25).to(dtype)
    sign = 1.0 - 2.0 * (torch.arange(n, device=dev) % 2)
    v = (sign[:, None, None] * torch.ones((n, n_kv, D), device=dev)).to(dtype)
    c, o, plan, ref = _step(dev, n_q, n_kv, past, new, k, v, dtype)
    q = torch.randn((sum(new), n_q, D), generator=g, device=dev).to(dtype)
    want, bound = o.attend(_np(q), ref, D ** -0.5)
    _check_attend(c.attend(0, q, plan), want, bound, dtype)


@pytest.mark.parametrize("new", [1, 3, 40])
def test_small_values_beside_large_ones_in_bf16_queries(dev, new):
    """A query's largest value meets keys of 0; the scores come from one 2^-18
    and one 2^-27 times as large, whose eight bits all count."""
    print(f"[bf16 query] {new}", flush=True)
    g = torch.Generator(device=dev).manual_seed(3)
    n_q, n_kv, past = 8, 2, 100
    n = past + new
    for small in (18, 27):
        k = torch.zeros((n, n_kv, D), device=dev)
        k[:, :, 1] = torch.randint(-7, 8, (n, n_kv), generator=g, device=dev) * 64.0
        v = torch.randn((n, n_kv, D), generator=g, device=dev).bfloat16()
        c, o, plan, ref = _step(dev, n_q, n_kv, [past], [new], k.bfloat16(), v, torch.bfloat16)
        q = torch.zeros((new, n_q, D), device=dev)
        q[..., 0] = 1.5
        q[..., 1] = (1 + torch.randint(0, 128, (new, n_q), generator=g, device=dev) / 128) * 2.0 ** -small
        q = q.bfloat16()
        scale = 2.0 ** (small - 8)
        want, bound = o.attend(_np(q), ref, scale)
        _check_attend(c.attend(0, q, plan, scale=scale), want, bound, torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_token_has_its_result_whatever_step_it_comes_in(dev, dtype):
    """Rows of a prompt against the same tokens in steps of one and of four, over
    the same cache: off by no more than two results of the same formula may be."""
    print(f"[steps] {dtype}", flush=True)
    g = torch.Generator(device=dev).manual_seed(4)
    n_q, n_kv, n = 8, 2, 90
    k, v = (torch.randn((n, n_kv, D), generator=g, device=dev).to(dtype) for _ in range(2))
    q = torch.randn((n, n_q, D), generator=g, device=dev).to(dtype)
    c, o, plan, ref = _step(dev, n_q, n_kv, [0], [n], k, v, dtype)
    whole = c.attend(0, q, plan)
    want, bound = o.attend(_np(q), ref, D ** -0.5)
    _check_attend(whole, want, bound, dtype)
    for t0, size in ((89, 1), (86, 4), (70, 1), (64, 4)):
        c.rewind([t0])
        p = c.extend([size], c.new_plan(size))
        y = c.attend(0, q[t0:t0 + size], p)       # the codes are still there
        _check_attend(y, want[t0:t0 + size], bound[t0:t0 + size], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("past,new", [(100000, 4096), (40000, 1)])
def test_many_small_weights_behind_a_large_one(dev, dtype, past, new):
    """One position 2^22 to 2^30 times as heavy as each of the others, whose
    values differ from its own: the others count together.  Where a workgroup
    has all of a row's pages (16 heads of 4096 tokens), a wave cuts every one of
    their weights; a weight's two parts end 2^-30 below the largest one."""
    print(f"[small weights] {dtype} {past} + {new}", flush=True)
    heads = 16
    k = torch.zeros((past, heads, D), device=dev, dtype=dtype)
    v = torch.ones_like(k)
    k[0, :, 0], v[0] = 1.0, -1.0
    c = oi2.PagedKVCache(1, heads, heads, 1, past + new, P.pages_of(past + new), device=dev)
    c.append(0, k, v, c.extend([past], c.new_plan(past)))
    plan = c.extend([new], c.new_plan(new))
    c.append(0, torch.zeros((new, heads, D), device=dev, dtype=dtype), torch.ones((new, heads, D), device=dev, dtype=dtype), plan)
    q = torch.zeros((new, heads, D), device=dev, dtype=dtype)
    for bits in (22, 24, 25, 25.5, 26, 26.5, 27, 28, 30):
        q[:, :, 0] = bits * np.log(2)
        gap = q[0, 0, 0].item()
        y = _np(c.attend(0, q, plan, scale=1.0)[[0, -1]])
        for t, out in ((0, y[0]), (new - 1, y[1])):
            w = (past + t) * np.exp(-gap)
            want = (w - 1) / (w + 1)
            # half a step; the cut, of every weight; fp32: a score of up to 44 in
            # powers of two, 2^-18, and an exponential's and a sum's few steps
            # of the small weights
            tol = torch.finfo(dtype).eps / 2 * abs(want) + (past + t) * 2.0 ** -30 + 2 * w * 2.0 ** -17
            assert np.abs(out - want).max() <= tol, (bits, t, np.abs(out - want).max() / tol)


@pytest.mark.parametrize("new", [1, 40])
def test_scores_past_fp32_beside_scores_of_zero(dev, new):
    """A query and a key whose product passes fp32: minus infinity weighs nothing,
    and the other positions, whose keys are 0, share the rest."""
    print(f"[large scores] {new}", flush=True)
    past, n_q, n_kv = 70, 4, 2
    n = past + new
    k = torch.zeros((n, n_kv, D), device=dev)
    k[3, :, 0] = -2.0 ** 60
    v = torch.randint(-7, 8, (n, n_kv, D), generator=torch.Generator(device=dev).manual_seed(6), device=dev).float()
    c, o, plan, ref = _step(dev, n_q, n_kv, [past], [new], k.bfloat16(), v.bfloat16(), torch.bfloat16)
    q = torch.zeros((new, n_q, D), device=dev)
    q[..., 0] = 2.0 ** 100
    y = _np(c.attend(0, q.bfloat16(), plan, scale=1.0))
    v = _np(v)
    for t in range(new):
        seen = np.delete(v[:past + t + 1], 3, 0)
        for h in range(n_q):
            x = seen[:, h // (n_q // n_kv)]
            tol = 2.0 ** -8 * np.abs(x.mean(0)) + P.attend_bound(0.0, 0.0, n, False) * np.abs(x).mean(0)
            assert (np.abs(y[t, h] - x.mean(0)) <= tol).all()
