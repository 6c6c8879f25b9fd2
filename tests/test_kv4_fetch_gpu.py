"""Positions of a 4-bit cache read back: outputs that are slices of one buffer,
as many rows as a cache may have, more pages than workgroups, rooms much larger
than what is read, groups that are not finite.  Bit for bit against the float64
oracle; bf16 is its fp32 value, exact, rounded by torch.
"""
import ctypes
import itertools
import math
import random

import numpy as np
import pytest
import torch

import oi2
from oi2 import _lib
from tests.test_gpu_paged import _extend, _np, _values, dev  # noqa: F401
from tests.test_kv4_gpu import _held, _pair

pytestmark = pytest.mark.gpu
D = 128


def _want(x, dtype, dev):
    return torch.from_numpy(x).to(torch.float32).to(dtype).to(dev)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("n_kv", [1, 3, 8])
def test_fetch_into_slices_of_one_buffer(dev, dtype, n_kv):
    """Every order of k and v, tokens and heads, with 16-byte stores and without,
    k and v exchanged; what lies between and behind the values is kept."""
    print(f"[fetch4 one buffer] {dtype} kv {n_kv}", flush=True)
    c, o = _held(dev, n_kv, [100, 33], torch.float16)
    first, count, n, room = [0, 5], [100, 20], 120, 131
    k, v, cu = o.fetch(first, count)
    want = [_want(x, dtype, dev) for x in (k, v)]
    size = {"kv": 2, "t": room, "h": n_kv}
    for gap, order, swap in itertools.product((0, 8, 1), itertools.permutations(["kv", "t", "h"]), (0, 1)):
        one = torch.full([size[d] for d in order] + [D + gap], 5.0, dtype=dtype, device=dev)
        outs = one.permute([order.index(d) for d in ("kv", "t", "h")] + [3])[..., :D]
        a, b = outs[swap], outs[1 - swap]
        ka, va, gcu = c.fetch(0, count, room, first=first, dtype=dtype, k_out=a, v_out=b)
        assert ka is a and va is b and gcu.tolist() == cu
        assert torch.equal(a[:n], want[0]) and torch.equal(b[:n], want[1]), (gap, order, swap)
        assert bool((outs[:, n:] == 5).all()) and bool((one[..., D:] == 5).all())


def _check_fetch(c, o, first, count, rooms, dev, dtypes=(torch.float16, torch.float32, torch.bfloat16)):
    k, v, cu = o.fetch(first, count)
    f, n = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (first, count))
    for dtype in dtypes:
        want = [_want(x, dtype, dev) for x in (k, v)]
        for room in rooms:
            *got, gcu = c.fetch(0, n, room, first=f, dtype=dtype)
            assert gcu.tolist() == cu
            m = min(cu[-1], room)
            for x, y in zip(got, want):
                assert torch.equal(x[:m], y[:m]) and not x[m:].any(), (dtype, room)


@pytest.mark.parametrize("n_seqs", [64, 65, 127, 128, 200, 255, 256, 257, 700, 2047, 2048])
def test_fetch_of_many_rows(dev, n_seqs):
    """Sums over several waves, and over several rows a thread: empty rows, rows
    left out, ranges inside rows and past their ends."""
    print(f"[fetch4 rows] {n_seqs}", flush=True)
    rng = random.Random(n_seqs)
    most = 150 if n_seqs < 300 else 9
    lens = [rng.choice([0, 1, 3, rng.randint(0, most)]) for _ in range(n_seqs)]
    lens[rng.randrange(n_seqs)] = 130
    lens[-1] = 70
    c, o = _held(dev, 2, lens, torch.float16, seed=n_seqs)
    for first, count in (([0] * n_seqs, lens), ([rng.randint(-1, n // 2 + 1) for n in lens], [rng.randint(-1, n + 2) for n in lens]),
                         ([0] * n_seqs, [0] * (n_seqs - 1) + [70]), ([0] * n_seqs, [n if i % 64 == 63 else 0 for i, n in enumerate(lens)])):
        total = o.fetch(first, count)[2][-1]
        _check_fetch(c, o, first, count, sorted({0, 1, total // 2, max(total - 1, 0), total, total + 37}), dev,
                     (torch.float16,) if n_seqs % 64 else (torch.float16, torch.bfloat16))


@pytest.mark.parametrize("n_kv,lens", [(32, [2200, 1500, 0, 900]), (12, [6400, 64, 5000, 1]), (1, [100000, 40000])])
def test_fetch_of_more_pages_than_workgroups(dev, n_kv, lens):
    """2048 workgroups at most, which take several pages of a head each."""
    print(f"[fetch4 pages] kv {n_kv} {lens}", flush=True)
    g = torch.Generator(device=dev).manual_seed(n_kv)
    pages = sum(-(-n // 64) for n in lens)
    assert pages * n_kv > 2048
    c, _ = _pair(n_kv, len(lens), max(lens), pages, dev, n_q=n_kv, shuffle=n_kv)
    plan = c.extend(lens, c.new_plan(sum(lens)))
    k, v = (_values(g, (sum(lens), n_kv, D), torch.float16, dev) for _ in range(2))
    c.append(0, k, v, plan)
    # what codes and scales say of each position, in the rows' order
    at = torch.cat([c.block_table[i, torch.arange(n, device=dev) // 64].long() * 64 + torch.arange(n, device=dev) % 64 for i, n in enumerate(lens)])
    want = []
    for codes, scales in zip(c.codes(0), c.scales(0)):
        x = codes.float() * scales.reshape(pages, n_kv, 64, 4).float().repeat_interleave(32, 3)
        want.append(x.transpose(1, 2).reshape(pages * 64, n_kv, D)[at])
    for first in (0, 40):
        held = torch.cat([torch.arange(n, device=dev) >= first for n in lens])
        for dtype in (torch.float16, torch.bfloat16):
            *got, cu = c.fetch(0, lens, sum(lens), first=[first] * len(lens), dtype=dtype)
            n = int(held.sum())
            assert cu.tolist() == np.cumsum([0] + [max(m - first, 0) for m in lens]).tolist()
            for x, y in zip(got, want):
                assert torch.equal(x[:n], y[held].to(dtype)) and not x[n:].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_fetch_into_much_more_room(dev, dtype):
    """Rows past the last token: all of them 0, whatever the memory held, over
    many turns of every workgroup; none of them touched without the flag."""
    print(f"[fetch4 room] {dtype}", flush=True)
    room, n_kv = 20000, 8
    c, o = _held(dev, n_kv, [70, 5], torch.float16)
    k, v, cu = o.fetch([3, 0], [60, 5])
    count, first = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([60, 5], [3, 0]))
    outs = [torch.full((room, n_kv, D), math.nan, dtype=dtype, device=dev) for _ in range(2)]
    gcu = torch.full((3,), -1, dtype=torch.int32, device=dev)
    hk, hv = (_lib.heads(x, n_kv)[1] for x in outs)
    lib, ref = oi2.load_library(), ctypes.byref
    for flag in (0, _lib.ZERO_LEFT_OUT):
        torch.cuda.synchronize()
        assert lib.oi2_kv4_fetch(c._ref, 0, first.data_ptr(), count.data_ptr(), _lib.dtype_code(dtype) | flag, room, ref(hk), ref(hv),
                                 gcu.data_ptr(), torch.cuda.current_stream(dev).cuda_stream or None) == 0
        assert gcu.tolist() == cu
        for x, y in zip(outs, (k, v)):
            assert torch.equal(x[:65], _want(y, dtype, dev))
            assert bool((x[65:] == 0).all()) if flag else bool(x[65:].isnan().all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_fetch_of_groups_that_are_not_finite(dev, dtype):
    """They are NaN in every type, their neighbours what they are without them;
    so are they in a row read back, and in the cache that they are moved to."""
    print(f"[fetch4 nan] {dtype}", flush=True)
    g = torch.Generator(device=dev).manual_seed(2)
    c, o = _pair(3, 2, 200, 5, dev, n_q=3)
    plan = c.new_plan(200)
    ref = _extend(c, o, plan, [130, 20])
    k, v = (_values(g, (150, 3, D), dtype, dev) for _ in range(2))
    for i, bad in enumerate((math.nan, math.inf, -math.inf)):
        k[40 * i + 7, i, 32 * i + 5], v[149 - 50 * i, 2 - i, 127 - 33 * i] = bad, bad
    k[64, 1, 0:128:32] = math.inf
    c.append(0, k, v, plan)
    o.append(_np(k), _np(v), ref)
    want = o.fetch([0, 0], [130, 20])[:2]
    assert [int(np.isnan(x).sum()) for x in want] == [32 * 7, 32 * 3]
    for to in (torch.float16, torch.float32, torch.bfloat16):
        for x, y in zip(c.fetch(0, [130, 20], 150, dtype=to), want):
            y = _want(y, to, dev)
            assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num())
    for x, y in zip(c.read(0, 0, torch.float32), o.held(0, 130)):
        assert np.array_equal(_np(x), y, equal_nan=True)
    fk, fv, _ = c.fetch(0, [130, 20], 150)
    c2, _ = _pair(3, 2, 200, 5, dev, n_q=3)
    c2.append(0, fk, fv, c2.extend([130, 20], c2.new_plan(150)))
    for x, y in zip(c2.fetch(0, [130, 20], 150), (fk, fv, None)):
        assert y is None or torch.equal(x.nan_to_num(), y.nan_to_num()) and torch.equal(x.isnan(), y.isnan())
