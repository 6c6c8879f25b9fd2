"""The paged 4-bit KV cache on the GPU against the float64 oracle: the codes that
a step leaves, positions read back, the attention, and the three as a layer and a
serving loop use them.

Codes, scales and what they stand for are compared bit for bit; attention outputs
may be off by half a step of their type and the oracle's bound on fp32 sums, on
the probabilities' two fp16 parts and on the smallest weights.
"""
import math
import random

import numpy as np
import pytest
import torch

import oi2
from oracle import oracle as O
from oracle import paged as P8
from oracle import paged4 as P
from tests.gpu_helpers import EPS, assert_ffn_close
from tests.test_gpu_attention import _cfg, _dense, _weights
from tests.test_gpu_paged import SCALINGS, _check_attend, _extend, _ints, _np, _values, dev  # noqa: F401

pytestmark = pytest.mark.gpu
D = 128
H, N_Q = 4096, 32
NAN = 0x7E00


def _pair(n_kv, n_seqs, max_len, n_pages, dev, n_q=N_Q, layers=1, shuffle=None):
    c = oi2.PagedKVCache(layers, n_q, n_kv, n_seqs, max_len, n_pages, device=dev, bits=4)
    o = P.Cache4(n_seqs, max_len, n_pages, n_kv)
    if shuffle is not None:
        order = list(range(n_pages))
        random.Random(shuffle).shuffle(order)
        c.free.copy_(torch.tensor(order, dtype=torch.int32))
        o.free = list(order)
    return c, o


def _same(x, y):
    differ = ~((x == y) | (np.isnan(x) & np.isnan(y)))
    assert not differ.any(), f"{differ.sum()} differ, the first at {np.argwhere(differ)[0]}: {x[differ][0]}, not {y[differ][0]}"


def _check_codes(c, o, layer=0):
    for got, scale, codes, scales in zip(c.codes(layer), c.scales(layer), o.codes, o.scales):
        assert got.dtype == torch.int8 and scale.dtype == torch.float16
        _same(got.cpu().numpy().astype(np.float64), codes)
        _same(_np(scale.reshape(c.n_pages, c.n_kv, 64, 4)), scales)


# ── append ───────────────────────────────────────────────────────────────────

STEPS = [
    (4, [[1, 64, 65, 0], [1, 1, 1, 1], [63, 0, 70, 5], [1, 200, 1, 64]]),
    (2, [[0, 3], [130, 1], [1, 60], [1, 1], [64, 64]]),
    (1, [[1]] * 3 + [[61]] + [[1], [190]]),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n_kv", [1, 3, 8, 32])
@pytest.mark.parametrize("n_seqs,steps", STEPS)
def test_append_codes(dev, dtype, n_kv, n_seqs, steps):
    """Pages growing over several steps, of values of every size."""
    print(f"[append4] {dtype} kv {n_kv} rows {n_seqs}", flush=True)
    g = torch.Generator(device=dev).manual_seed(n_kv)
    c, o = _pair(n_kv, n_seqs, 500, 24, dev, n_q=n_kv, shuffle=1)
    plan = c.new_plan(300)
    for i, new in enumerate(steps):
        ref = _extend(c, o, plan, new)
        n = sum(new)
        k = _values(g, (n, n_kv, D), dtype, dev) * [1.0, 40.0, 0.01, 3000.0, 1e-6, 1.0][i]
        v = _values(g, (n, n_kv, D), dtype, dev) * [1.0, 0.01, 40.0, 1e-5, 300.0, 1.0][i]
        k, v = k.clamp(-6e4, 6e4), v.clamp(-6e4, 6e4)
        assert c.append(0, k, v, plan) is None
        o.append(_np(k), _np(v), ref)
        _check_codes(c, o)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_special_values(dev, dtype):
    """Zeros, subnormals, the type's largest and lowest, infinities and NaN; ties
    between codes under every scale of 8 bits, and ties of the scales."""
    c, o = _pair(2, 3, 600, 40, dev, n_q=2)
    plan = c.new_plan(700)
    f = torch.finfo(dtype)
    inf = math.inf
    special = torch.tensor([0.0, -0.0, f.tiny, f.smallest_normal / 8, f.max, f.min, inf, -inf, math.nan, 1.0], dtype=torch.float64)
    for step, (new, scale) in enumerate([([0, 1, 20], 0.0), ([5, 5, 44], 1.0), ([260, 2, 300], 1.0)]):
        ref = _extend(c, o, plan, new)
        n = sum(new)
        g = torch.Generator().manual_seed(step)
        k, v = (torch.randn((n, 2, D), generator=g, dtype=torch.float64) * scale for _ in range(2))
        if step == 1:
            for j, s in enumerate(special):            # each in a group of its own
                k[j, 0, 3], v[j + 10, 1, 127] = s, s
            k[20, 0, :10], v[20, 0, :10] = special, special
            k[21] = 0.0
            v[22, 1, 32:64] = -0.0
            k[23] = f.max
            v[23] = f.min
        if step == 2:
            # scale m 2^e with m of 8 bits, each code's midpoint to the next one: m (2 j + 1) 2^(e - 1), which 11 bits hold
            # for the smaller m; the largest value 7 m 2^e
            m = 128 + torch.arange(n, dtype=torch.float64) % 128
            e = torch.tensor([-20.0, -7.0, 0.0, 5.0])[torch.arange(n) % 4].double()
            unit = (m * 2.0 ** e)[:, None, None]
            j = torch.arange(-6, 7, dtype=torch.float64)
            k[:, :, :13] = unit * (j + 0.5)
            k[:, :, 13] = 7 * unit[..., 0]
            k[:, :, 14:32] = 0.0
            # the scale's own ties: top = 7 (m + 1/2) 2^e
            v[:, 1, 64:96] = 0.0
            v[:, 1, 70] = -(7 * (m + 0.5)) * 2.0 ** e
            k, v = k.clamp(-6e4, 6e4), v.clamp(-6e4, 6e4)
        k, v = k.to(dtype).to(dev), v.to(dtype).to(dev)
        c.append(0, k, v, plan)
        o.append(_np(k), _np(v), ref)
        _check_codes(c, o)


def test_append_every_fp16_value(dev):
    """Every finite fp16 value as the largest of its group, and as another beside
    a largest of 1 to 2^8 times it."""
    c, o = _pair(8, 1, 4096, 64, dev, n_q=8)
    plan = c.new_plan(4096)
    g = torch.Generator().manual_seed(1)
    x = torch.arange(0x7C00, dtype=torch.int16).view(torch.float16).double()
    x = torch.cat([x, torch.zeros(32768 - x.numel(), dtype=torch.float64)])
    k = x.reshape(1024, 8, 4, 1) * torch.rand((1024, 8, 4, 32), generator=g, dtype=torch.float64)
    k[..., 7] = -x.reshape(1024, 8, 4)
    v = x.reshape(1024, 8, 4, 1) * (2 * torch.rand((1024, 8, 4, 32), generator=g, dtype=torch.float64) - 1)
    v[..., 31] = (x.reshape(1024, 8, 4) * 2.0 ** (torch.arange(1024) % 9)[:, None, None]).clamp(max=65504)
    k, v = (y.reshape(1024, 8, D).half().to(dev) for y in (k, v))
    ref = _extend(c, o, plan, [1024])
    c.append(0, k, v, plan)
    o.append(_np(k), _np(v), ref)
    _check_codes(c, o)


@pytest.mark.parametrize("dtype,layout,part", [
    (torch.float16, "half", 128), (torch.bfloat16, "interleaved", 64), (torch.float16, "half", 50), (torch.bfloat16, "half", 96),
    (torch.float16, "interleaved", 2), (torch.bfloat16, "half", 16), (torch.float16, "interleaved", 128), (torch.bfloat16, "half", 2),
    (torch.float16, "interleaved", 90)])
def test_append_is_rotary_and_append(dev, dtype, layout, part):
    """The fused call gives the bits of the two: q, codes and scales; with any
    strides, in pages that grow, tokens of rejected rows left out."""
    print(f"[append4 rotary] {dtype} {layout} {part}", flush=True)
    g = torch.Generator(device=dev).manual_seed(part)
    rot = oi2.Rotary(D, 5e5, rotary_dim=part, layout=layout, device=dev, scaling=SCALINGS[4] if part > 60 else SCALINGS[0])
    a, b = (oi2.PagedKVCache(2, 32, 8, 5, 400, 20, device=dev, bits=4) for _ in range(2))
    pa, pb = a.new_plan(500), b.new_plan(500)
    for new in ([3, 70, 0, 129, 64], [1, 1, 1, 1, 1], [64, 0, 401, 5, 2]):
        a.extend(new, pa)
        b.extend(new, pb)
        n = sum(new)
        qkv = _values(g, (n, 48, D), dtype, dev)
        q, k, v = qkv[:, :32], qkv[:, 32:40], qkv[:, 40:]
        qo = torch.full((n, 32, D), 3.0, dtype=dtype, device=dev)
        assert a.append(1, k, v, pa, q=q, rotary=rot, q_out=qo) is qo
        q2, k2 = torch.full_like(qo, 3.0), torch.zeros_like(k.contiguous())
        rot(q, k, pb.positions[:n], q_out=q2, k_out=k2)
        odd = torch.empty((n, 8, D + 1), dtype=dtype, device=dev)[..., :D]
        odd.copy_(k2)
        b.append(1, odd, v.transpose(0, 1).contiguous().transpose(0, 1), pb)
        assert torch.equal(qo, q2)
        assert torch.equal(a.pages, b.pages)
        # k and v at odd addresses, q in place, k alone rotated: the same
        odd.copy_(k)
        qc = q.contiguous()
        assert b.append(1, odd, v, pb, q=qc, rotary=rot, q_out=qc) is qc
        assert torch.equal(a.pages, b.pages) and torch.equal(qc[pb.positions[:n] >= 0], q2[pb.positions[:n] >= 0])
        assert b.append(1, k, v, pb, rotary=rot) is None
        assert torch.equal(a.pages, b.pages)
    assert not a.pages[0].any()


def test_append_leaves_other_places(dev):
    """Places that the step does not write keep their bytes, those of tokens past
    the call's, of rejected rows and of slots outside the pool among them."""
    c, _ = _pair(2, 3, 300, 12, dev, n_q=2)
    plan = c.new_plan(200)
    c.pages.copy_(torch.randint(0, 256, c.pages.shape, device=dev, dtype=torch.uint8))
    before = [x.clone() for x in (*c.codes(0), *(y.contiguous().view(torch.int16) for y in c.scales(0)))]
    c.extend([5, 130, 301], plan)
    assert plan.rejected.tolist() == [0, 0, 1]
    k, v = (torch.randn(200, 2, D, device=dev).half() for _ in range(2))
    slots = plan.slots[:120].long()
    plan.slots[3], plan.slots[60] = 12 * 64, 2 ** 31 - 1            # damaged
    c.append(0, k[:120], v[:120], plan)
    slots[3] = slots[60] = slots[4]
    written = torch.zeros(12 * 64, dtype=torch.bool, device=dev)
    written[slots[slots >= 0]] = True
    after = [*c.codes(0), *(y.contiguous().view(torch.int16) for y in c.scales(0))]
    for x, y in zip(before, after):
        x, y = (t.reshape(12, 2, 64, -1).transpose(1, 2).reshape(12 * 64, 2, -1) for t in (x, y))
        assert torch.equal(x[~written], y[~written])
        assert not torch.equal(x[written], y[written])


# ── fetch ────────────────────────────────────────────────────────────────────

def _held(dev, n_kv, lens, dtype, seed=5, n_extra=2):
    g = torch.Generator(device=dev).manual_seed(seed)
    n_pages = sum(P8.pages_of(n) for n in lens) + n_extra
    c, o = _pair(n_kv, len(lens), max(max(lens), 1), n_pages, dev, n_q=n_kv, shuffle=seed)
    plan = c.new_plan(max(sum(lens), 1))
    ref = _extend(c, o, plan, lens)
    k, v = (_values(g, (sum(lens), n_kv, D), dtype, dev) for _ in range(2))
    if sum(lens):
        c.append(0, k, v, plan)
        o.append(_np(k), _np(v), ref)
    return c, o


@pytest.mark.parametrize("n_kv", [1, 3, 8, 32])
@pytest.mark.parametrize("lens,first,count", [
    ([1], [0], [1]), ([70], [0], [70]), ([70], [63], [2]), ([300, 0, 64, 129], [0, 0, 0, 0], [300, 5, 64, 129]),
    ([300, 10, 64, 129], [299, 10, 3, 60], [1, 7, 60, 80]), ([50, 60], [-5, 70], [20, 3]), ([50, 60], [20, 0], [-1, 2 ** 31 - 1]),
    ([40] * 33, list(range(33)), [3] * 33), ([0, 0], [0, 0], [4, 4]),
])
def test_fetch(dev, n_kv, lens, first, count):
    print(f"[fetch4] kv {n_kv} {lens[:4]} {first[:4]} {count[:4]}", flush=True)
    c, o = _held(dev, n_kv, lens, torch.float16)
    k, v, cu = o.fetch(first, count)
    n = cu[-1]
    for dtype in (torch.float16, torch.float32, torch.bfloat16):
        for room in {n, n + 9, max(n - 3, 0)}:
            gk, gv, gcu = c.fetch(0, count, room, first=first, dtype=dtype)
            assert gcu.tolist() == cu
            m = min(n, room)
            for got, want in ((gk, k), (gv, v)):
                assert got.shape == (room, n_kv, D) and got.dtype == dtype
                want = torch.from_numpy(want[:m]).to(dtype if dtype != torch.bfloat16 else torch.float32).to(dtype)
                assert torch.equal(got[:m].cpu(), want)
                assert not got[m:].any()
    assert torch.equal(c.fetch(0, count, n)[2].cpu(), torch.tensor(np.cumsum([0] + [min(max(a, 0), b) for a, b in zip(count, lens)])).int())


@pytest.mark.parametrize("room", [0, 1, 36, 37, 38, 64, 100, 101, 137, 138, 400])
def test_fetch_of_more_than_there_is_room_for(dev, room):
    """Rooms that end in a row, at its end, on a page's edge and inside a page,
    where rows start inside one."""
    print(f"[fetch4] room {room}", flush=True)
    c, o = _held(dev, 3, [101, 64, 0, 200], torch.float16)
    first, count = [27, 0, 0, 63], [37, 64, 9, 2 ** 31 - 1]
    k, v, cu = o.fetch(first, count)
    gk, gv, gcu = c.fetch(0, count, room, first=first)
    assert gcu.tolist() == cu
    m = min(cu[-1], room)
    for got, want in ((gk, k), (gv, v)):
        assert torch.equal(got[:m].cpu(), torch.from_numpy(want[:m]).half()) and not got[m:].any()


def test_fetch_is_what_read_gives(dev):
    c, o = _held(dev, 8, [130, 7, 0], torch.bfloat16)
    for row in (0, 1, 2, -2):
        k, v = c.read(0, row, torch.float32)
        wk, wv = o.held(row % 3, o.lens[row % 3])
        assert np.array_equal(_np(k), wk) and np.array_equal(_np(v), wv)
    assert c.read(0, 0)[0].dtype == torch.float16


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_fetch_into_given_outputs(dev, dtype):
    """Heads first as a dense cache has them, slices of one tensor, odd addresses;
    rows past the last token are kept."""
    c, o = _held(dev, 4, [100, 33], torch.float16)
    n = 133
    k, v, cu = c.fetch(0, [100, 33], n, dtype=dtype)
    heads_first = [torch.full((4, 150, D), 5.0, dtype=dtype, device=dev) for _ in range(2)]
    one = torch.full((150, 9, D), 5.0, dtype=dtype, device=dev)
    odd = [torch.full((150, 4, D + 1), 5.0, dtype=dtype, device=dev) for _ in range(2)]
    for a, b in (tuple(x.transpose(0, 1) for x in heads_first), (one[:, :4], one[:, 5:]), (one[:, 5:], one[:, :4]),
                 tuple(x[..., 1:] for x in odd)):
        ka, va, _ = c.fetch(0, [100, 33], 150, dtype=dtype, k_out=a, v_out=b)
        assert ka is a and va is b
        assert torch.equal(a[:n], k) and torch.equal(b[:n], v) and bool((a[n:] == 5).all()) and bool((b[n:] == 5).all())
    assert bool((one[:, 4] == 5).all()) and all(bool((x[..., 0] == 5).all()) for x in odd)


def test_fetch_refusals(dev):
    c, _ = _held(dev, 4, [20], torch.float16)
    x = torch.zeros((8, 4, D), dtype=torch.float16, device=dev)
    bad = [(ValueError, (0, [1, 2], 4), {}), (ValueError, (0, [1], -1), {}), (ValueError, (1, [1], 4), {}), (TypeError, (0, [1], 4), {"dtype": torch.int8}),
           (ValueError, (0, [1], 8), {"k_out": x}), (ValueError, (0, [1], 4), {"k_out": x, "v_out": x}),
           (ValueError, (0, [1], 8), {"k_out": x, "v_out": x.float()}), (ValueError, (0, [1], 8), {"k_out": x, "v_out": x.cpu()}),
           (oi2.OI2Error, (0, [1], 8), {"k_out": x, "v_out": x}), (oi2.OI2Error, (0, [1], 8), {"k_out": x, "v_out": x[:1].expand(8, 4, D)}),
           (ValueError, (0, [1], 4), {"first": [1, 2]})]
    for err, args, kw in bad:
        with pytest.raises(err):
            c.fetch(*args, **kw)
    with pytest.raises(ValueError):
        oi2.PagedKVCache(1, 8, 8, 1, 64, 1, device=dev).fetch(0, [1], 4)


def test_fetch_moves_requests_to_another_cache(dev):
    """A prefix leaves one cache and enters another: what it stands for is coded
    to what it stands for (its largest value is 7 of its scale)."""
    a, _ = _held(dev, 8, [200, 77, 3], torch.float16)
    k, v, cu = a.fetch(0, [150, 77, 0], 300)
    b, _ = _pair(8, 2, 400, 9, dev, n_q=8)
    plan = b.extend([150, 77], b.new_plan(300))
    assert torch.equal(plan.cu, cu[:3])
    b.append(0, k, v, plan)
    k2, v2, _ = b.fetch(0, [150, 77], 300)
    assert torch.equal(k, k2) and torch.equal(v, v2)


# ── attention ────────────────────────────────────────────────────────────────

def _filled(dev, n_q, n_kv, past, new, dtype, seed, max_new=None, n_extra=3, layers=1):
    g = torch.Generator(device=dev).manual_seed(seed)
    n_pages = sum(P8.pages_of(a + b) for a, b in zip(past, new)) + n_extra
    c, o = _pair(n_kv, len(past), max(max(a + b for a, b in zip(past, new)), 1), n_pages, dev, n_q=n_q, shuffle=seed, layers=layers)
    # whatever the pool's pages held before: NaN scales, any codes
    c.pages.copy_(torch.randint(0, 256, c.pages.shape, device=dev, dtype=torch.uint8))
    first = c.new_plan(max(sum(past), 1))
    plan = c.new_plan(max(sum(new), 1), max_new=max_new or max(max(new), 1))
    for p, lens in ((first, past), (plan, new)):
        ref = _extend(c, o, p, lens)
        k, v = (_values(g, (sum(lens), n_kv, D), dtype, dev) for _ in range(2))
        if sum(lens):
            c.append(layers - 1, k, v, p)
            o.append(_np(k), _np(v), ref)
    q = torch.randn((sum(new), n_q, D), generator=g, device=dev).to(dtype)
    return c, o, plan, ref, q


CASES = [
    # past, new
    ([0], [1]), ([63], [1]), ([64], [1]), ([255], [1]), ([1000], [1]), ([5000], [1]),
    ([3, 700, 64, 0, 1281], [1, 1, 1, 1, 1]),
    ([3, 700, 64, 0, 1281], [1, 0, 1, 0, 1]),
    ([0, 100, 2000], [2, 1, 4]),
    ([10, 300], [3, 16]),
    ([0], [64]), ([0], [65]), ([0], [33]), ([0], [200]),
    ([100, 0, 1500], [100, 31, 1]),
    ([3000, 40], [40, 1]),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("past,new", CASES)
def test_attend(dev, dtype, past, new):
    for n_kv in ((1, 8) if len(past) > 1 else (8, 32)):
        n_q = 8 if n_kv == 1 else 32
        print(f"[attend4] {dtype} {past} {new} q {n_q} kv {n_kv}", flush=True)
        c, o, plan, ref, q = _filled(dev, n_q, n_kv, past, new, dtype, 7)
        want, bound = o.attend(_np(q), ref, D ** -0.5)
        _check_attend(c.attend(0, q, plan), want, bound, dtype)


@pytest.mark.parametrize("n_q,n_kv", [(1, 1), (2, 1), (4, 1), (8, 1), (32, 16), (12, 3)])
def test_attend_head_layouts(dev, n_q, n_kv):
    print(f"[attend4] heads {n_q} {n_kv}", flush=True)
    for past, new in (([70, 900], [1, 1]), ([70, 300], [5, 150])):
        c, o, plan, ref, q = _filled(dev, n_q, n_kv, past, new, torch.float16, 3)
        want, bound = o.attend(_np(q), ref, D ** -0.5)
        _check_attend(c.attend(0, q, plan), want, bound, torch.float16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [[1, 1, 1], [2, 40, 300], [8, 5, 7], [16, 9, 7]])
def test_attend_values_of_many_sizes(dev, dtype, new):
    """Groups whose k and v differ by many powers of two, all-zero ones among
    them, and other scales of the scores: 0, negative, large."""
    print(f"[attend4 sizes] {dtype} {new}", flush=True)
    g = torch.Generator(device=dev).manual_seed(2)
    past, n_kv, n_q = [640, 513, 100], 4, 16
    n_pages = sum(P8.pages_of(a + b) for a, b in zip(past, new))
    c, o = _pair(n_kv, 3, 1000, n_pages, dev, n_q=n_q, shuffle=9)
    first, plan = c.new_plan(sum(past)), c.new_plan(sum(new))
    for p, lens in ((first, past), (plan, new)):
        ref = _extend(c, o, p, lens)
        n = sum(lens)
        k, v = (_values(g, (n, n_kv, D), dtype, dev) for _ in range(2))
        at = torch.arange(n, device=dev)[:, None, None] * 31 + torch.arange(D, device=dev) // 32 * 7
        v = (v.double() * torch.exp2(at % 23 - 11.0)).clamp(-6e4, 6e4).to(dtype)
        v[at.expand(v.shape) % 5 == 3] = 0.0
        k = (k.double() * torch.exp2(at % 5 - 2.0)).to(dtype)
        c.append(0, k, v, p)
        o.append(_np(k), _np(v), ref)
    q = torch.randn((sum(new), n_q, D), generator=g, device=dev).to(dtype)
    for scale in (0.02, 0.0, -0.03, 0.4):
        want, bound = o.attend(_np(q), ref, float(np.float32(scale)))
        _check_attend(c.attend(0, q, plan, scale=scale), want, bound, dtype)


@pytest.mark.parametrize("new", [[1, 1], [3, 2], [90, 150], [7, 8], [16, 11]])
def test_attend_nan_where_it_is_seen(dev, new):
    """A group of v that is not finite reaches the rows that see its position, in
    its dims alone; one of k the rows that see it, in every dim; none what lies
    behind, whatever freed pages still hold."""
    print(f"[attend4 nan] {new}", flush=True)
    g = torch.Generator(device=dev).manual_seed(4)
    past, n_kv, n_q = [130, 64], 2, 8
    c, o = _pair(n_kv, 2, 400, 9, dev, n_q=n_q)
    first, plan = c.new_plan(600), c.new_plan(sum(new))
    # pages full of NaN, given back to the pool
    c.extend([300, 250], first)
    bad = torch.full((550, n_kv, D), math.nan, device=dev).half()
    c.append(0, bad, bad, first)
    c.rewind([0, 0])
    o.extend([300, 250], 600, 600)
    o.rewind([0, 0])
    for step, (p, lens) in enumerate(((first, past), (plan, new))):
        ref = _extend(c, o, p, lens)
        k, v = (_values(g, (sum(lens), n_kv, D), torch.float16, dev) for _ in range(2))
        if step == 0:
            v[10, 0, 64] = math.inf                       # by every later token of row 0, in a page that all see
        if step == 1:
            v[sum(new) - 1, 1, 7] = math.nan              # seen by the last token alone
            v[new[0] // 2, 0, 100] = math.inf             # by the later half of row 0
            if new[0] > 1:
                k[new[0] - 1, 1, 3] = math.nan            # by row 0's last token
        c.append(0, k, v, p)
        o.append(_np(k), _np(v), ref)
    q = torch.randn((sum(new), n_q, D), generator=g, device=dev).half()
    want, bound = o.attend(_np(q), ref, D ** -0.5)
    nan = np.isnan(want)
    assert nan.any() and not nan.all()
    _check_attend(c.attend(0, q, plan), want, bound, torch.float16)


@pytest.mark.parametrize("n_kv,past,new", [(8, [20000], [1]), (8, [9000, 300, 5000], [1, 1, 1]), (8, [6000], [300]),
                                           (4, [7000, 20, 4000], [2, 250, 1]), (8, [9000, 300, 5000], [8, 5, 7]),
                                           (4, [6000, 900], [4, 3]), (4, [6000, 900], [7, 8])])
def test_attend_rows_cut_into_parts(dev, n_kv, past, new):
    print(f"[attend4 parts] kv {n_kv} {past} + {new}", flush=True)
    c, o, plan, ref, q = _filled(dev, 32, n_kv, past, new, torch.float16, 11)
    want, bound = o.attend(_np(q), ref, D ** -0.5)
    y = c.attend(0, q, plan)
    _check_attend(y, want, bound, torch.float16)
    for _ in range(3):
        assert torch.equal(c.attend(0, q, plan), y)


@pytest.mark.parametrize("n_q,n_kv,new", [(32, 8, [8, 5, 6, 7]), (32, 8, [9, 8, 33, 40]), (32, 4, [3, 4, 5, 2]), (8, 8, [17, 31, 32, 33]),
                                          (4, 2, [16, 9, 17, 8]), (4, 2, [16, 9, 13, 8]), (32, 8, [16, 9, 12, 3]), (32, 4, [8, 5, 7, 6]),
                                          (8, 8, [33, 64, 1, 49]), (8, 8, [65, 64, 1, 49]), (8, 8, [17, 31, 32, 5]), (32, 8, [8, 1, 6, 3]),
                                          (32, 4, [3, 4, 1, 2])])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend_tiles_around_17_to_64_rows(dev, dtype, n_q, n_kv, new):
    """Drafts, and ends of chunks: more rows than one set, up to two and four of
    them, one beyond; cut into parts and not; calls with fewer tokens than the plan's."""
    for past in ([0, 63, 64, 200], [1500, 10, 2000, 1100]):
        print(f"[attend4 sets] {dtype} q {n_q} kv {n_kv} {past} + {new}", flush=True)
        c, o, plan, ref, q = _filled(dev, n_q, n_kv, past, new, dtype, 17)
        want, bound = o.attend(_np(q), ref, D ** -0.5)
        y = c.attend(0, q, plan)
        _check_attend(y, want, bound, dtype)
        assert torch.equal(c.attend(0, q, plan), y)
        for n in (1, new[0] - 1, new[0], new[0] + 1, sum(new) - 1):
            got = c.attend(0, q[:n], plan)
            _check_attend(got, want[:n], bound[:n], dtype)


def test_attend_every_position_counts_once(dev):
    """Values that name their position, so that one lost or doubled at an edge of
    pages, parts or tiles shows: scores of 0, so that the result is the mean."""
    for n_kv, n in ((8, 1), (1, 16), (8, 40)):
        for length in (1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1025, 1100):
            print(f"[attend4 positions] kv {n_kv} new {n} length {length}", flush=True)
            total = length + n
            c, o = _pair(n_kv, 1, total, P8.pages_of(total), dev, n_q=8)
            plan = c.new_plan(total)
            ref = _extend(c, o, plan, [total])
            k = torch.zeros((total, n_kv, D), device=dev).half()
            pos = torch.arange(total, device=dev)
            v = (7.0 * ((pos[:, None] >> (torch.arange(D, device=dev) % 11)) & 1))[:, None].expand(-1, n_kv, -1).half()
            c.append(0, k, v, plan)
            c.rewind([length])
            step = c.extend([n], c.new_plan(n))
            c.append(0, k[length:], v[length:], step)
            q = torch.ones((n, 8, D), device=dev).half()
            y = _np(c.attend(0, q, step))
            bits = ((np.arange(total)[:, None] >> (np.arange(D) % 11)) & 1).astype(np.float64)
            sums = np.cumsum(bits, 0)[length:] * 7 / np.arange(length + 1, total + 1)[:, None]
            # half a step of fp16; sums and the division in fp32, weights of 2^6 exact
            assert (np.abs(y - sums[:, None]) <= (2.0 ** -11 + 2.0 ** -20) * sums[:, None]).all()


def test_attend_strides_outputs_and_first_tokens(dev):
    c, o, plan, ref, q = _filled(dev, 32, 8, [70, 900, 5], [3, 1, 40], torch.bfloat16, 13)
    y = c.attend(0, q, plan)
    want, bound = o.attend(_np(q), ref, D ** -0.5)
    _check_attend(y, want, bound, torch.bfloat16)
    odd = torch.empty((44, 32, D + 1), dtype=q.dtype, device=dev)[..., :D]
    odd.copy_(q)
    for x in (q.transpose(0, 1).contiguous().transpose(0, 1), odd):
        assert torch.equal(c.attend(0, x, plan), y)
    x = q.clone()
    assert c.attend(0, x, plan, out=x) is x and torch.equal(x, y)
    for n in (0, 1, 3, 4, 30):
        assert torch.equal(c.attend(0, q[:n], plan), y[:n])


def test_attend_rejected_rows_and_padding(dev):
    c, o = _pair(8, 3, 100, 3, dev)
    plan = c.new_plan(60)
    c.extend([50, 101, 1], plan)
    assert plan.rejected.tolist() == [0, 1, 1]          # a rejected row keeps its tokens: the last one ends past 60
    c2 = oi2.PagedKVCache(1, 32, 8, 3, 300, 9, device=dev, bits=4)
    p2 = c2.extend([50, 8, 1], c2.new_plan(60, max_new=50))
    n = 60
    k, v = (torch.randn((n, 8, D), device=dev).half() for _ in range(2))
    q = torch.randn((n, 32, D), device=dev).half()
    c2.append(0, k, v, p2)
    y = c2.attend(0, q, p2)
    assert y[:59].any(2).all() and not y[59:].any()
    given = torch.full_like(q, 9.0)
    c2.attend(0, q, p2, out=given)
    assert torch.equal(given[:59], y[:59]) and bool((given[59:] == 9).all())
    p3 = c2.extend([1, 500, 1], c2.new_plan(600, max_new=600))
    c2.append(0, k[:2], v[:2], p3)
    z = c2.attend(0, q, p3)
    assert z[0].any() and not z[1:].any()


@pytest.mark.parametrize("max_new", [4, 8, 16, 40])
def test_attend_rejected_rows_with_many_tokens(dev, max_new):
    """Rows with more tokens than the plan's rows may have keep them in the packed
    order, and get zeros there whichever tiles they are in."""
    print(f"[attend4 rejected] {max_new}", flush=True)
    new = [max_new, 200, 3, max_new + 1, 1]
    c = oi2.PagedKVCache(1, 32, 8, 5, 400, 30, device=dev, bits=4)
    plan = c.extend(new, c.new_plan(sum(new) + 5, max_new=max_new))
    assert plan.rejected.tolist() == [0, 1, 0, 1, 0]
    n = sum(new)
    k, v = (torch.randn((n, 8, D), device=dev).half() for _ in range(2))
    c.append(0, k, v, plan)
    q = torch.randn((n + 5, 32, D), device=dev).half()
    y = torch.full_like(q, 9.0)
    c.attend(0, q, plan, out=y)
    at = np.cumsum([0] + new)
    for i, rejected in enumerate([0, 1, 0, 1, 0]):
        x = y[at[i]:at[i + 1]]
        assert not x.any() if rejected else bool((x != 9).any(2).all()) and bool(x.any(2).all())
    assert bool((y[n:] == 9).all())


# ── together ─────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("n_kv", [8, 32])
@pytest.mark.parametrize("past,new", [([5], [1]), ([200, 64, 7], [1, 1, 1]), ([3000, 70], [1, 1]), ([2500, 1300], [7, 130]), ([1800], [8]), ([0, 130, 63, 9, 1], [1, 2, 0, 1, 1]),
                                      ([0, 300], [70, 1]), ([40, 0, 100], [3, 190, 1])])
def test_layer_over_pages(dev, n_kv, past, new):
    """GroupedQueryAttention.forward_paged: the pages are append's of the same
    projections, the output the float64 chain's over what they stand for."""
    print(f"[paged4 layer] kv {n_kv} {past} + {new}", flush=True)
    g = torch.Generator(device=dev).manual_seed(11)
    w = _weights(dev, n_kv, seed=12)
    rows, n_pages = len(past), sum(P8.pages_of(a + b) for a, b in zip(past, new))
    attn = oi2.GroupedQueryAttention(0, w, _cfg(n_kv))
    rot = oi2.Rotary(D, 1e4, device=dev)
    most = max(400, *(a + b for a, b in zip(past, new)))
    c, c2 = (oi2.PagedKVCache(2, N_Q, n_kv, rows, most, n_pages, device=dev, bits=4) for _ in range(2))
    o = P.Cache4(rows, most, n_pages, n_kv)
    wq, _, _, wo, nw = _dense(w)
    one, zero = torch.ones((4000, D // 2), device=dev), torch.zeros((4000, D // 2), device=dev)
    for step in (past, new):
        n = sum(step)
        plan, p2 = (x.extend(step, x.new_plan(n + 3, max_new=max(step))) for x in (c, c2))
        ref = o.extend(step, n + 3, max(step))
        x = torch.randn((n + 3, H), generator=g, device=dev).half()
        resid = torch.empty_like(x)
        out = attn.forward_paged(x, c, plan, rot, layer=1, residual_out=resid)
        assert torch.equal(resid, (x.float() + out.float()).half())
        assert not out[n:].any()
        # counters of parts are cleared whatever the workspace's memory held; the step is coded again, to the same
        dirty = torch.full((64 << 20,), 255, dtype=torch.uint8, device=dev)
        del dirty
        assert torch.equal(attn.forward_paged(x, c, plan, rot, layer=1), out)
        _, (k, v) = oi2.GroupedQueryAttention(0, w, _cfg(n_kv))(x[None], one, zero)
        c2.append(1, k[0].transpose(0, 1), v[0].transpose(0, 1), p2, rotary=rot)
        assert torch.equal(c.pages, c2.pages)
        for i, (codes, scale) in enumerate(zip(c.codes(1), c.scales(1))):
            o.codes[i] = codes.cpu().numpy().astype(np.float64)
            o.scales[i] = _np(scale.reshape(n_pages, n_kv, 64, 4))
        if not n:
            continue
        xn = O.f16(O.rmsnorm(x[:n].float().cpu().numpy().astype(np.float64), nw, EPS))
        q = O.f16(xn @ wq.T).reshape(n, N_Q, D)
        q = O.f16(P8.rotate(q, ref["positions"][:n], oi2.rotary_frequencies(D, 1e4)[0], 1.0, "half"))
        a = O.f16(o.attend(q, ref, D ** -0.5)[0]).reshape(n, H)
        assert_ffn_close(out[:n].float().cpu().numpy(), O.f16(a @ wo.T), what="paged layer")


def test_serving_loop_captured(dev):
    """Steps of extend, append, attend and fetch captured once and replayed over
    growing rows, with eager work between, against the same calls made eagerly."""
    print("[kv4 graph]", flush=True)
    g = torch.Generator(device=dev).manual_seed(17)
    rot = oi2.Rotary(D, 1e4, device=dev)
    caches = [oi2.PagedKVCache(1, N_Q, 8, 4, 3000, 160, device=dev, bits=4) for _ in range(2)]
    prompt = [1500, 63, 0, 700]
    qkv = torch.randn((sum(prompt), 48, D), generator=g, device=dev).half()
    plans = []
    for c in caches:
        p = c.extend(prompt, c.new_plan(sum(prompt)))
        c.append(0, qkv[:, 32:40], qkv[:, 40:], p, rotary=rot)
        plans.append(c.new_plan(4, max_new=1))
    new = torch.tensor([1, 1, 1, 1], dtype=torch.int32, device=dev)
    first = torch.tensor([1490, 0, 0, 650], dtype=torch.int32, device=dev)
    count = torch.tensor([20, 64, 2, 60], dtype=torch.int32, device=dev)
    x = torch.zeros((4, 48, D), dtype=torch.float16, device=dev)

    def step(c, plan, x):
        c.extend(new, plan)
        q = c.append(0, x[:, 32:40], x[:, 40:], plan, q=x[:, :32], rotary=rot)
        return (c.attend(0, q, plan), *c.fetch(0, count, 160, first=first))

    stream = torch.cuda.Stream(device=dev)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    before = [t.clone() for t in (caches[0].lens, caches[0].block_table, caches[0].free, caches[0].n_free)]
    with torch.cuda.graph(graph, stream=stream):
        outs = step(caches[0], plans[0], x)
    for a, b in zip(before, (caches[0].lens, caches[0].block_table, caches[0].free, caches[0].n_free)):
        assert torch.equal(a, b)                        # capturing runs nothing
    for i in range(70):
        x.copy_(torch.randn((4, 48, D), generator=g, device=dev))
        graph.replay()
        got = [t.clone() for t in outs]
        want = step(caches[1], plans[1], x)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), f"replay {i}"
        for t in outs:
            t.zero_()
    assert torch.equal(caches[0].pages, caches[1].pages)


@pytest.mark.parametrize("past,new", [([9000, 300, 5000], [1, 1, 1]), ([7000, 20, 4000], [2, 250, 1]), ([9000, 300, 5000], [8, 1, 5])])
def test_layers_of_a_step_on_two_streams(dev, past, new):
    """attend and fetch of two layers at the same time."""
    print(f"[kv4 streams] {past} + {new}", flush=True)
    g = torch.Generator(device=dev).manual_seed(3)
    c = oi2.PagedKVCache(2, N_Q, 8, 3, 10000, 400, device=dev, bits=4)
    first = c.extend(past, c.new_plan(sum(past)))
    plan = c.new_plan(sum(new), max_new=max(new))
    for li in range(2):
        x = torch.randn((sum(past), 16, D), generator=g, device=dev).half()
        c.append(li, x[:, :8], x[:, 8:], first)
    c.extend(new, plan)
    for li in range(2):
        x = torch.randn((sum(new), 16, D), generator=g, device=dev).half()
        c.append(li, x[:, :8], x[:, 8:], plan)
    q = [torch.randn((sum(new), N_Q, D), generator=g, device=dev).half() for _ in range(2)]
    count = torch.tensor([100, 300, 50], dtype=torch.int32, device=dev)

    def both(li):
        return (c.attend(li, q[li], plan), *c.fetch(li, count, 450))
    want = [both(li) for li in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for li, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[li].append(both(li))
    torch.cuda.synchronize()
    for li in range(2):
        for y in got[li]:
            assert all(torch.equal(a, b) for a, b in zip(y, want[li]))


def test_pools_past_4_gb(dev):
    """The last pages of a pool whose offsets pass 32 bits."""
    n_pages = 70000                                     # 5.2 GB
    c = oi2.PagedKVCache(1, 32, 8, 2, 300, n_pages, device=dev, bits=4)
    o = P.Cache4(2, 300, 10, 8)
    c.free.copy_(torch.arange(n_pages, dtype=torch.int32, device=dev))      # the last pages first
    plan = c.new_plan(400, max_new=200)
    c.extend([200, 150], plan)
    ref = o.extend([200, 150], 400, 200)
    assert int(c.block_table[0, 0]) == n_pages - 1
    k, v = (torch.randn((350, 8, D), device=dev).half() for _ in range(2))
    q = torch.randn((350, 32, D), device=dev).half()
    c.append(0, k, v, plan)
    o.append(_np(k), _np(v), ref)
    fk, fv, _ = c.fetch(0, [200, 150], 350)
    wk, wv, _ = o.fetch([0, 0], [200, 150])
    assert np.array_equal(_np(fk), wk) and np.array_equal(_np(fv), wv)
    want, bound = o.attend(_np(q), ref, D ** -0.5)
    _check_attend(c.attend(0, q, plan), want, bound, torch.float16)
    assert _ints(c.lens).tolist() == [200, 150]
