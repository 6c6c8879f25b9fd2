"""The append of short steps (plans of up to eight new tokens a row): codes and
scales bit for bit against the oracle, for both types, layouts, parts of the head
and strides, with pages that grow at every edge of their groups of positions."""
import math

import pytest
import torch

import oi2
from tests.test_gpu_paged import _check_codes, _extend, _np, _pair, _values, dev  # noqa: F401

pytestmark = pytest.mark.gpu
D = 128
# what rows hold before the first step: every edge of a page and of its groups of 16
PAST = [0, 1, 14, 15, 16, 17, 31, 47, 62, 63, 64, 65]
ROPES = [None, ("half", 128), ("half", 96), ("half", 50), ("half", 2), ("interleaved", 128), ("interleaved", 64), ("interleaved", 6)]


def _strided(x, how):
    if how == "heads first":
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    if how == "odd":
        y = torch.empty((*x.shape[:2], D + 1), dtype=x.dtype, device=x.device)[..., 1:]
        return y.copy_(x)
    return x


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("max_new", [1, 4, 8])
@pytest.mark.parametrize("rope", ROPES)
def test_codes_of_short_steps(dev, dtype, max_new, rope):
    print(f"[append few] {dtype} {max_new} {rope}", flush=True)
    g = torch.Generator(device=dev).manual_seed(max_new)
    n_kv, rows = 3, len(PAST)
    rot = rope and oi2.Rotary(D, 1e4, rotary_dim=rope[1], layout=rope[0], device=dev)
    c, o = _pair(n_kv, rows, 128, 2 * rows, dev, n_q=n_kv, shuffle=2)
    first = c.new_plan(sum(PAST))
    ref = _extend(c, o, first, PAST)
    k, v = (_values(g, (sum(PAST), n_kv, D), dtype, dev, 0.2) for _ in range(2))
    c.append(0, k, v, first)
    o.append(_np(k), _np(v), ref)
    _check_codes(c, o)
    plan = c.new_plan(max_new * rows, max_new=max_new)
    # k's and v's scales grow at different steps, by few and by many powers of two, or not
    for i, (mk, mv, how) in enumerate(((1.0, 1.0, ""), (2.0 ** 5, 2.0 ** -6, "odd"), (2.0 ** -9, 2.0 ** 4, "heads first"),
                                       (2.0 ** 10, 2.0 ** 11, "odd"), (1.0, 1.0, "heads first"))):
        new = [1 + (r + i) % max_new if (r + i) % 5 else 0 for r in range(rows)]
        ref = _extend(c, o, plan, new)
        n = sum(new)
        k, v = _strided(_values(g, (n, n_kv, D), dtype, dev, 0.2) * mk, how), _strided(_values(g, (n, n_kv, D), dtype, dev, 0.2) * mv, how)
        c.append(0, k, v, plan, rotary=rot)
        # a key is rounded to its type before it is coded: the rotary's own bits
        turned = rot(k, None, plan.positions[:n])[0] if rot else k
        o.append(_np(turned), _np(v), ref)
        _check_codes(c, o)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("held", [0, 1, 15, 16, 17, 63])
def test_special_values(dev, dtype, held):
    """Zeros, subnormals, the type's extremes, infinities and NaN, ties between
    codes, the largest value at the edge of a scale, in a page that holds ``held``
    positions; then a step that grows what holds a NaN."""
    print(f"[append few] special {dtype} held {held}", flush=True)
    f = torch.finfo(dtype)
    c, o = _pair(4, 1, 200, 4, dev, n_q=4)
    if held:
        plan = c.new_plan(held)
        ref = _extend(c, o, plan, [held])
        x = torch.linspace(-1, 1, held * 4 * D, device=dev).view(held, 4, D).to(dtype)
        c.append(0, x, x.flip(2), plan)
        o.append(_np(x), _np(x.flip(2)), ref)
    plan = c.new_plan(8, max_new=8)
    special = torch.tensor([0.0, -0.0, f.tiny, f.smallest_normal / 8, f.max, f.min, math.inf, -math.inf, math.nan, 1.0], dtype=torch.float64)
    e = torch.arange(127, dtype=torch.float64)
    val = torch.where(e < 8, e * 2.0 ** -9, (1 + (e % 8) / 8) * 2.0 ** (e // 8 - 7))
    ties = (val[:-1] + val[1:]) / 2
    for step in range(4):
        n = (1, 8, 3, 5)[step]
        k, v = (torch.zeros(n, 4, D, dtype=torch.float64) for _ in range(2))
        if step == 0:
            k[:, 0, :126], v[:, 1, :126] = ties, -ties            # under a largest value of 448
            k[:, 0, 127] = v[:, 1, 127] = 448.0
        elif step == 1:
            k[3, 0, 20:30], v[5, 1, 70:80] = special, special
            k[0, 2], v[7, 3] = 448.0, 1.75
            k[2, 2, 9] = 448.5 if dtype == torch.float16 else 450.0
        elif step == 2:
            k[:, 1], v[:, 0] = f.max, f.min                       # grows what holds a NaN, of v's head 1 not
            v[0, 1] = f.max
        k, v = k.to(dtype).to(dev), v.to(dtype).to(dev)
        ref = _extend(c, o, plan, [n])
        c.append(0, k, v, plan)
        o.append(_np(k), _np(v), ref)
        _check_codes(c, o)
    used = c.block_table[0, :2].long()
    used = used[used >= 0]
    bad = torch.isnan(c.codes(0)[1].contiguous().view(c.n_pages, 4, 64 * D).float()).any(-1)[used]
    assert torch.equal(c.scales(0)[1][used] < 0, bad)
