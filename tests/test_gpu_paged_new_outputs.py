"""New outputs of the paged operators hold no old memory: tokens without a
position (of rejected rows, past the step's last one, at negative positions) have
0 there.  Outputs that the caller gives keep those rows."""
import math

import pytest
import torch

import oi2
from tests.test_gpu_paged import dev  # noqa: F401

pytestmark = pytest.mark.gpu
D = 128
DTYPES = [torch.float16, torch.bfloat16]


def _stain(like):
    """What the next tensor of this size finds in its memory."""
    for _ in range(3):
        torch.full_like(like, math.nan, memory_format=torch.contiguous_format)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout,part", [("half", 128), ("interleaved", 50)])
def test_rotary(dev, dtype, layout, part):
    rot = oi2.Rotary(D, 1e4, rotary_dim=part, layout=layout, device=dev)
    for n in (5, 700):
        print(f"[new outputs] rotary {dtype} {layout} {part} {n}", flush=True)
        q, k = (torch.randn(n, h, D, device=dev).to(dtype) for h in (4, 2))
        pos = torch.arange(n, device=dev, dtype=torch.int32)
        out = pos % 3 == 1
        pos = torch.where(out, -1 - pos, pos)
        for x in (q, k):
            _stain(x)
        y, z = rot(q, k, pos)
        full = rot(q, k, pos.abs())
        for a, b in ((y, full[0]), (z, full[1])):
            assert (a[out] == 0).all() and torch.equal(a[~out], b[~out])
        # one output given: it keeps its rows, the new one has zeros
        given = torch.full_like(q, 7.0)
        _stain(k)
        y, z = rot(q, k, pos, q_out=given)
        assert y is given and (y[out] == 7.0).all() and (z[out] == 0).all() and torch.equal(y[~out], full[0][~out])
        given = torch.full_like(k, 7.0)
        _stain(q)
        y, z = rot(q, k, pos, k_out=given)
        assert z is given and (z[out] == 7.0).all() and (y[out] == 0).all() and torch.equal(z[~out], full[1][~out])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,n,max_new", [([1, 1, 1, 0], 7, 1), ([3, 0, 2, 1], 9, 3), ([40, 1, 200, 30], 300, None), ([5, 1, 0, 0], 2000, None)])
def test_append_and_attend(dev, dtype, new, n, max_new):
    """Row 2 rejected: the pool has no page for it."""
    print(f"[new outputs] step {dtype} {new} of {n}", flush=True)
    rot = oi2.Rotary(D, 1e4, device=dev)
    c = oi2.PagedKVCache(1, 8, 2, 4, 256, 4, device=dev)
    c.append(0, *(torch.randn(92, 2, D, device=dev).to(dtype) for _ in range(2)), c.extend([10, 10, 64, 8], c.new_plan(92)))
    plan = c.new_plan(n, max_new=max_new)
    q = torch.randn(n, 8, D, device=dev).to(dtype)
    k, v = (torch.randn(n, 2, D, device=dev).to(dtype) for _ in range(2))
    # before the first step no token has a position
    _stain(q)
    assert not c.append(0, k, v, plan, q=q, rotary=rot).any()
    _stain(q)
    assert not c.attend(0, q, plan).any()
    c.extend(new, plan)
    live = plan.positions[:n] >= 0
    assert plan.rejected[2] == (1 if new[2] else 0) and live.any() and not live.all()
    _stain(q)
    y = c.append(0, k, v, plan, q=q, rotary=rot)
    assert not y[~live].any() and y[live].any()
    assert torch.equal(y[live], rot(q, None, plan.positions[:n])[0][live])
    _stain(q)
    z = c.attend(0, y, plan)
    assert not z[~live].any() and z[live].flatten(1).any(1).all()
    given = torch.full_like(q, 9.0)
    c.attend(0, y, plan, out=given)
    assert torch.equal(given[live], z[live]) and (given[sum(new):] == 9.0).all()


def test_in_place_rows_stay(dev):
    rot = oi2.Rotary(D, 1e4, device=dev)
    c = oi2.PagedKVCache(1, 8, 2, 2, 64, 1, device=dev)
    plan = c.extend([2, 1], c.new_plan(5))
    q = torch.randn(5, 8, D, device=dev).half()
    before = q.clone()
    k = torch.randn(5, 2, D, device=dev).half()
    assert c.append(0, k, k, plan, q=q, rotary=rot, q_out=q) is q
    assert torch.equal(q[2:], before[2:]) and torch.equal(q[:2], rot(before, None, plan.positions)[0][:2])
