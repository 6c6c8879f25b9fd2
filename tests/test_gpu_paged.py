"""The paged 8-bit KV cache on the GPU against the float64 oracle: tables and
slot maps, rotary positions, the quantising append, the attention.

Tables, codes and scales are compared bit for bit.  Rotary outputs may be off
by half a step of their type and of fp32, and the pair times 2^-40 (fp64 on both sides) and
times what half a step of a 64-bit frequency makes at the token's position; attention outputs by half a step of their type
and the oracle's bound on fp32 sums and on the probabilities' fp16 parts (two
for fp16 outputs of up to 16 query rows, otherwise one).
"""
import math
import random

import numpy as np
import pytest
import torch

import oi2
from oracle import paged as P

pytestmark = pytest.mark.gpu
D = 128
N_Q = 32


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a visible GPU"
    return torch.device("cuda:0")


def _np(x):
    return x.detach().float().cpu().numpy().astype(np.float64)


def _ints(x):
    return x.cpu().numpy().astype(np.int64)


def _pair(n_kv, n_seqs, max_len, n_pages, dev, n_q=N_Q, layers=1, shuffle=None):
    c = oi2.PagedKVCache(layers, n_q, n_kv, n_seqs, max_len, n_pages, device=dev)
    o = P.Cache(n_seqs, max_len, n_pages, n_kv)
    if shuffle is not None:
        order = list(range(n_pages))
        random.Random(shuffle).shuffle(order)
        c.free.copy_(torch.tensor(order, dtype=torch.int32))
        o.free = list(order)
    return c, o


def _check_tables(c, o):
    assert _ints(c.lens).tolist() == list(o.lens)
    assert np.array_equal(_ints(c.block_table), o.table)
    n = int(c.n_free)
    assert n == len(o.free)
    assert _ints(c.free)[:n].tolist() == [int(x) for x in o.free]


def _extend(c, o, plan, new):
    c.extend(new, plan)
    ref = o.extend(new, plan.max_tokens, plan.max_new)
    assert _ints(plan.cu).tolist() == ref["cu"]
    assert _ints(plan.kv_len).tolist() == ref["kv_len"]
    assert _ints(plan.rejected).tolist() == ref["rejected"]
    assert np.array_equal(_ints(plan.positions), ref["positions"])
    assert np.array_equal(_ints(plan.slots), ref["slots"])
    _check_tables(c, o)
    return ref


def _values(g, shape, dtype, dev, spread=0.7):
    x = torch.randn(shape, generator=g, device=dev) * torch.exp(spread * torch.randn(shape[1:], generator=g, device=dev))
    return x.to(dtype)


def _check_codes(c, o, layer=0):
    for got, scale, codes, exps in zip(c.codes(layer), c.scales(layer), o.codes, o.exps):
        x = got.contiguous().view(c.n_pages, c.n_kv, 64, 128).float().cpu().numpy()
        assert np.array_equal(_np(scale.abs()), 2.0 ** exps.astype(np.float64))
        assert np.array_equal(np.isnan(x), np.isnan(codes))
        assert np.array_equal(np.nan_to_num(x), np.nan_to_num(codes))


def _check_attend(out, ref, bound, dtype, rows=None):
    y = _np(out)[:ref.shape[0]]
    assert np.array_equal(np.isnan(y), np.isnan(ref))
    tol = torch.finfo(dtype).eps / 2 * np.abs(ref) + 1.01 * bound + 2.0 ** -25
    err = np.abs(np.nan_to_num(y - ref))
    worst = (err / np.nan_to_num(tol, nan=1.0)).max() if err.size else 0.0
    assert worst <= 1.0, f"off by {worst:.3f} of the bound"


# ── tables ───────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("n_seqs,max_len,n_pages,max_tokens,max_new,steps", [
    (1, 64, 1, 64, 64, 6),
    (3, 200, 9, 40, 40, 12),
    (17, 1000, 60, 300, 150, 25),        # runs out of pages again and again
    (64, 129, 100, 64, 3, 30),
    (300, 700, 900, 2000, 700, 12),
    (1025, 300, 2500, 5000, 200, 8),     # positions in a launch of their own
    (2048, 90, 4096, 4097, 90, 6),
])
def test_tables_and_slots(dev, n_seqs, max_len, n_pages, max_tokens, max_new, steps):
    rng = random.Random(n_seqs)
    c, o = _pair(8, n_seqs, max_len, n_pages, dev, layers=0, shuffle=5)
    plan = c.new_plan(max_tokens, max_new=max_new)
    for s in range(steps):
        print(f"[paged tables] rows {n_seqs} step {s}", flush=True)
        top = max(1, 2 * max_tokens // n_seqs)
        new = [rng.choice([0, 0, 1, rng.randint(0, top), rng.randint(0, min(max_new + 2, 64)), -rng.randint(0, 3)])
               for _ in range(n_seqs)]
        _extend(c, o, plan, new)
        to = [rng.choice([-1, -1, 0, n, n + 5, max(n - rng.randint(0, 70), 0)]) for n in o.lens]
        c.rewind(to)
        o.rewind(to)
        _check_tables(c, o)


def test_extend_and_rewind_undo_each_other(dev):
    c, o = _pair(8, 9, 500, 40, dev, layers=0, shuffle=3)
    plan = c.new_plan(600)
    _extend(c, o, plan, [3, 64, 65, 0, 128, 1, 200, 7, 63])
    before = [x.clone() for x in (c.lens, c.block_table, c.free, c.n_free)]
    lens = c.lens.clone()
    c.extend([70, 1, 0, 300, 64, 2, 5, 60, 2], plan)
    c.rewind(lens)
    for x, y in zip(before, (c.lens, c.block_table, c.free, c.n_free)):
        assert torch.equal(x, y)


def test_lengths_past_every_size(dev):
    """Sums of lengths past 32 bits, rows past the buffer and past max_len."""
    c, o = _pair(8, 5, 1000, 30, dev, layers=0)
    plan = c.new_plan(500)
    _extend(c, o, plan, [100, 2000, 5, 600, 1])
    c.extend([1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 2], plan)
    assert _ints(plan.rejected).tolist() == [0, 1, 1, 1, 1]
    assert _ints(plan.cu).tolist() == [0, 1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1]


# ── rotary ───────────────────────────────────────────────────────────────────

SCALINGS = [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
            {"type": "wavelength", "factor": 8.0, "original_len": 8192, "low_factor": 1.0, "high_factor": 4.0},
            {"type": "yarn", "factor": 16.0, "original_len": 4096, "beta_fast": 32.0, "beta_slow": 1.0}]


def _check_rotary(x, y, pos, rot):
    freqs, mag = oi2.rotary_frequencies(rot.rotary_dim, 10000.0, rot._scaling)
    ref = P.rotate(_np(x), pos, freqs, mag, rot.layout)
    pair = mag * np.abs(_np(x)).max(-1, keepdims=True) * 2
    angle = 2.0 ** -40 + 2 * math.pi * 2.0 ** -65 * np.array(pos, np.float64)[:, None, None]
    tol = (torch.finfo(x.dtype).eps / 2 + 2.0 ** -24) * np.abs(ref) + angle * pair + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    assert (np.abs(_np(y) - ref) <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("head_dim,part,tokens,n_q,n_kv,scaling", [
    (128, 128, 1, 32, 8, 0), (128, 64, 7, 32, 8, 1), (128, 96, 33, 8, 1, 2), (128, 32, 300, 3, 3, 3),
    (64, 64, 5, 4, 4, 4), (256, 128, 9, 2, 1, 0), (128, 2, 3, 5, 2, 0), (80, 50, 17, 3, 1, 1), (128, 128, 1000, 32, 8, 4),
])
def test_rotary(dev, dtype, layout, head_dim, part, tokens, n_q, n_kv, scaling):
    print(f"[rotary] {dtype} {layout} {head_dim} {part} {tokens}", flush=True)
    g = torch.Generator(device=dev).manual_seed(tokens)
    rot = oi2.Rotary(head_dim, 10000.0, rotary_dim=part, layout=layout, scaling=SCALINGS[scaling], device=dev)
    rot._scaling = SCALINGS[scaling]
    qkv = _values(g, (tokens, n_q + 2 * n_kv, head_dim), dtype, dev)
    q, k = qkv[:, :n_q], qkv[:, n_q:n_q + n_kv]
    pos = torch.randint(0, 200000, (tokens,), generator=g, device=dev, dtype=torch.int32)
    pos[0] = 2 ** 31 - 1 if tokens > 1 else 0
    a, b = rot(q, k, pos)
    n = min(tokens, 40)
    _check_rotary(q[:n], a[:n], pos[:n].tolist(), rot)
    _check_rotary(k[:n], b[:n], pos[:n].tolist(), rot)
    # any strides, in place and without k: the same bits
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty((tokens, n_q, head_dim + 1), dtype=dtype, device=dev)[..., :head_dim]
    odd.copy_(q)
    for x in (heads_first, odd, q.contiguous()):
        assert torch.equal(rot(x, None, pos)[0], a)
    x = q.contiguous()
    assert rot(x, None, pos, q_out=x)[0] is x and torch.equal(x, a)


def test_rotary_leaves_out_negative_positions(dev):
    rot = oi2.Rotary(128, 10000.0, device=dev)
    q = torch.randn(6, 4, 128, device=dev).half()
    out = torch.full_like(q, 7.0)
    pos = torch.tensor([0, -1, 5, -1, -2147483648, 9], dtype=torch.int32, device=dev)
    rot(q, None, pos, q_out=out)
    assert (out[[1, 3, 4]] == 7.0).all()
    assert torch.equal(out[0], q[0])
    assert not (out[[2, 5]] == 7.0).any()
    rot(q[:0], None, pos[:0])


# ── append ───────────────────────────────────────────────────────────────────

STEPS = [
    (4, [[1, 64, 65, 0], [1, 1, 1, 1], [63, 0, 70, 5], [1, 200, 1, 64]]),
    (2, [[0, 3], [130, 1], [1, 60], [1, 1], [64, 64]]),
    (1, [[1]] * 3 + [[61]] + [[1], [190]]),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n_kv", [1, 8, 32])
@pytest.mark.parametrize("n_seqs,steps", STEPS)
def test_append_codes(dev, dtype, n_kv, n_seqs, steps):
    """Pages growing over several steps, each step's values larger or smaller."""
    print(f"[append] {dtype} kv {n_kv} rows {n_seqs}", flush=True)
    g = torch.Generator(device=dev).manual_seed(n_kv)
    c, o = _pair(n_kv, n_seqs, 500, 24, dev, n_q=n_kv, shuffle=1)
    plan = c.new_plan(300)
    for i, new in enumerate(steps):
        ref = _extend(c, o, plan, new)
        n = sum(new)
        k = _values(g, (n, n_kv, D), dtype, dev) * [1.0, 40.0, 0.01, 3000.0, 1e-6, 1.0][i]
        v = _values(g, (n, n_kv, D), dtype, dev) * [1.0, 0.01, 40.0, 1e-5, 300.0, 1.0][i]
        assert c.append(0, k, v, plan) is None
        o.append(_np(k), _np(v), ref)
        _check_codes(c, o)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_special_values(dev, dtype):
    """Zeros, subnormals, the type's largest and lowest, infinities and NaN; ties
    between codes; the largest value at the edge of a scale."""
    c, o = _pair(2, 3, 200, 9, dev, n_q=2)
    plan = c.new_plan(200)
    f = torch.finfo(dtype)
    inf = math.inf
    special = torch.tensor([0.0, -0.0, f.tiny, f.smallest_normal / 8, f.max, f.min, inf, -inf, math.nan, 1.0], dtype=torch.float64)
    for step, (new, scale) in enumerate([([0, 1, 20], 0.0), ([5, 5, 44], 1.0), ([64, 2, 30], 2.0)]):
        ref = _extend(c, o, plan, new)
        n = sum(new)
        g = torch.Generator().manual_seed(step)
        k, v = (torch.randn((n, 2, D), generator=g, dtype=torch.float64) * scale for _ in range(2))
        if step == 1:
            k[:, 0, :10], v[:, 1, :10] = special, special
            k[0, 1] = 448.0
            k[3, 1, 5] = 448.5 if dtype == torch.float16 else 450.0
            v[:, 0] = 0.0
        if step == 2:
            # every midpoint between neighbouring codes, under a largest value of 448
            e = torch.arange(127, dtype=torch.float64)
            val = torch.where(e < 8, e * 2.0 ** -9, (1 + (e % 8) / 8) * 2.0 ** (e // 8 - 7))
            mid = (val[:-1] + val[1:]) / 2
            k[:, :, :126], v[:, :, :126] = mid, -mid
        k, v = k.to(dtype).to(dev), v.to(dtype).to(dev)
        c.append(0, k, v, plan)
        o.append(_np(k), _np(v), ref)
        _check_codes(c, o)
    bad = torch.isnan(c.codes(0)[1].float()).flatten(2).any(-1)
    assert torch.equal(c.scales(0)[1] < 0, bad)


def test_append_is_rotary_and_append(dev):
    """The fused call gives the bits of the two: q, codes and scales; with any
    strides, in pages that grow, tokens of rejected rows left out."""
    for dtype, layout, part in ((torch.float16, "half", 128), (torch.bfloat16, "interleaved", 64), (torch.float16, "half", 50),
                                (torch.bfloat16, "half", 96), (torch.float16, "interleaved", 2)):
        print(f"[append rotary] {dtype} {layout} {part}", flush=True)
        g = torch.Generator(device=dev).manual_seed(part)
        rot = oi2.Rotary(D, 5e5, rotary_dim=part, layout=layout, device=dev, scaling=SCALINGS[3])
        a, b = (oi2.PagedKVCache(2, 32, 8, 5, 400, 20, device=dev) for _ in range(2))
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
            assert bool((a.pages == b.pages).all()) and bool((a._scales == b._scales).all())
        assert not a.pages[0].any() and not b.pages[0].any()


def test_append_leaves_other_places(dev):
    """Places that the step does not write keep their bytes."""
    c, _ = _pair(2, 2, 300, 12, dev, n_q=2)
    plan = c.new_plan(200)
    c.pages.copy_(torch.randint(0, 120, c.pages.shape, device=dev, dtype=torch.uint8))
    before = [x.contiguous().view(torch.uint8).clone() for x in c.codes(0)]
    c.extend([5, 130], plan)
    k, v = (torch.randn(135, 2, D, device=dev).half() for _ in range(2))
    c.append(0, k, v, plan)
    slots = plan.slots[:135].long()
    written = torch.zeros(12 * 64, dtype=torch.bool, device=dev)
    written[slots] = True
    for x, y in zip(before, (x.contiguous().view(torch.uint8) for x in c.codes(0))):
        x, y = (t.view(12, 2, 64, D).transpose(1, 2).reshape(12 * 64, 2, D) for t in (x, y))
        assert torch.equal(x[~written], y[~written])
        assert not torch.equal(x[written], y[written])


# ── attention ────────────────────────────────────────────────────────────────

def _filled(dev, n_q, n_kv, past, new, dtype, seed, max_new=None, n_extra=3, layers=1):
    """Caches (product and oracle) holding ``past``, a step of ``new`` appended
    after it, and its q."""
    g = torch.Generator(device=dev).manual_seed(seed)
    n_seqs = len(past)
    n_pages = sum(P.pages_of(a + b) for a, b in zip(past, new)) + n_extra
    c, o = _pair(n_kv, n_seqs, max(max(a + b for a, b in zip(past, new)), 1), n_pages, dev, n_q=n_q, shuffle=seed, layers=layers)
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
        print(f"[attend] {dtype} {past} {new} q {n_q} kv {n_kv}", flush=True)
        c, o, plan, ref, q = _filled(dev, n_q, n_kv, past, new, dtype, 7)
        want, bound = o.attend(_np(q), ref, D ** -0.5, q.dtype == torch.bfloat16)
        _check_attend(c.attend(0, q, plan), want, bound, dtype)


@pytest.mark.parametrize("n_q,n_kv", [(1, 1), (2, 1), (4, 1), (8, 1), (32, 16), (12, 3)])
def test_attend_head_layouts(dev, n_q, n_kv):
    print(f"[attend] heads {n_q} {n_kv}", flush=True)
    for past, new in (([70, 900], [1, 1]), ([70, 300], [5, 150])):
        c, o, plan, ref, q = _filled(dev, n_q, n_kv, past, new, torch.float16, 3)
        want, bound = o.attend(_np(q), ref, D ** -0.5, q.dtype == torch.bfloat16)
        _check_attend(c.attend(0, q, plan), want, bound, torch.float16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [[1, 1, 1], [2, 40, 300]])
def test_attend_pages_of_different_scales(dev, dtype, new):
    """Pages whose k and v differ by many powers of two, all-zero pages among
    them, and scores that rise and fall along the row."""
    print(f"[attend scales] {dtype} {new}", flush=True)
    g = torch.Generator(device=dev).manual_seed(2)
    past, n_kv, n_q = [640, 513, 100], 4, 16
    n_pages = sum(P.pages_of(a + b) for a, b in zip(past, new))
    c, o = _pair(n_kv, 3, 1000, n_pages, dev, n_q=n_q, shuffle=9)
    first, plan = c.new_plan(sum(past)), c.new_plan(sum(new))
    for p, lens in ((first, past), (plan, new)):
        ref = _extend(c, o, p, lens)
        n = sum(lens)
        k, v = (_values(g, (n, n_kv, D), dtype, dev) for _ in range(2))
        block = torch.arange(n, device=dev) // 64
        top = 10.0 if dtype == torch.float16 else 60.0
        v = (v.double() * torch.exp2(((block * 7919) % 23 - 11.0) / 11 * top)[:, None, None]).clamp(-6e4, 6e4).to(dtype)
        v[block % 5 == 3] = 0.0
        k = (k.double() * torch.exp2((block * 31) % 5 - 2.0)[:, None, None]).to(dtype)
        c.append(0, k, v, p)
        o.append(_np(k), _np(v), ref)
    q = torch.randn((sum(new), n_q, D), generator=g, device=dev).to(dtype)
    want, bound = o.attend(_np(q), ref, 0.02, q.dtype == torch.bfloat16)
    y = c.attend(0, q, plan, scale=0.02)
    if dtype == torch.float16:
        assert np.abs(want).max() < 6.5e4
    _check_attend(y, want, bound, dtype)


@pytest.mark.parametrize("new", [[1, 1], [3, 2], [90, 150]])
def test_attend_nan_where_it_is_seen(dev, new):
    """A NaN in v reaches the rows that see its position, in its dim alone; one
    in k the rows that see it, in every dim; none what lies behind, whatever
    freed pages still hold."""
    print(f"[attend nan] {new}", flush=True)
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
        if step == 1:
            v[sum(new) - 1, 1, 7] = math.nan              # seen by the last token alone
            v[new[0] // 2, 0, 100] = math.inf             # by the later half of row 0
            if new[0] > 1:
                k[new[0] - 1, 1, 3] = math.nan            # by row 0's last token
        c.append(0, k, v, p)
        o.append(_np(k), _np(v), ref)
    q = torch.randn((sum(new), n_q, D), generator=g, device=dev).half()
    want, bound = o.attend(_np(q), ref, D ** -0.5, q.dtype == torch.bfloat16)
    y = c.attend(0, q, plan)
    nan = np.isnan(want)
    assert nan.any() and not nan.all()
    _check_attend(y, want, bound, torch.float16)


def test_attend_zero_rows_of_rejected_and_untouched_rows(dev):
    c, o, plan, ref, q = _filled(dev, 32, 8, [100, 60, 5, 128], [1, 1, 1, 0], torch.float16, 1, max_new=1, n_extra=0)
    assert int(c.n_free) == 0
    plan = c.new_plan(6, max_new=2)
    c.extend([1, 4, 1, 0], plan)                 # row 1: past max_new
    assert plan.rejected.tolist() == [0, 1, 0, 0]
    k = torch.randn(6, 8, D, device=dev).half()
    c.append(0, k, k, plan)
    out = torch.full((6, 32, D), 9.0, device=dev).half()
    q = torch.randn(6, 32, D, device=dev).half()
    c.attend(0, q, plan, out=out)
    assert (out[1:5] == 0).all() and not (out[0] == 9.0).any() and not (out[5] == 9.0).any()
    # fewer tokens than the plan has room for: the rows behind the last one stay
    c.extend([1, 0, 1, 0], plan)
    out.fill_(9.0)
    c.append(0, k, k, plan)
    c.attend(0, q, plan, out=out)
    assert (out[2:] == 9.0).all() and not (out[:2] == 9.0).any()
    # no page left: row 0 has room in its own, row 1 and those behind it need one; row 3 is full
    plan = c.new_plan(70)
    c.extend([1, 4, 64, 1], plan)
    assert plan.rejected.tolist() == [0, 1, 1, 1]
    out = torch.full((70, 32, D), 9.0, device=dev).half()
    q = torch.randn(70, 32, D, device=dev).half()
    c.append(0, torch.zeros(70, 8, D, device=dev).half(), torch.zeros(70, 8, D, device=dev).half(), plan)
    c.attend(0, q, plan, out=out)
    assert (out[1:] == 0).all() and not (out[0] == 9.0).any()


def test_attend_strides_and_repeats(dev):
    """q with any strides, twice the same bits, another scale; scores of zero
    average the values."""
    c, o, plan, ref, q = _filled(dev, 32, 8, [700, 90, 3], [1, 20, 3], torch.bfloat16, 6)
    y = c.attend(0, q, plan)
    odd = torch.empty((24, 32, D + 1), dtype=q.dtype, device=dev)[..., :D]
    odd.copy_(q)
    for x in (odd, q.transpose(0, 1).contiguous().transpose(0, 1), q):
        assert torch.equal(c.attend(0, x, plan), y)
    want, bound = o.attend(_np(q), ref, 0.0, q.dtype == torch.bfloat16)
    _check_attend(c.attend(0, q, plan, scale=0.0), want, bound, torch.bfloat16)
    want, bound = o.attend(_np(q), ref, -0.3, q.dtype == torch.bfloat16)
    _check_attend(c.attend(0, q, plan, scale=-0.3), want, bound, torch.bfloat16)


def test_a_run_of_steps(dev):
    """Prompts, tokens, drafts, a roll back, a sequence's end and its row's next
    one, over two layers, the whole of it against the oracle."""
    g = torch.Generator(device=dev).manual_seed(0)
    n_kv, n_q, rows = 8, 32, 4
    rot = oi2.Rotary(D, 1e4, device=dev)
    c = oi2.PagedKVCache(2, n_q, n_kv, rows, 600, 30, device=dev)
    o = [P.Cache(rows, 600, 30, n_kv) for _ in range(2)]
    plan, small = c.new_plan(400), c.new_plan(16, max_new=4)
    steps = [(plan, [100, 0, 37, 200]), (small, [1, 0, 1, 1]), (small, [4, 4, 4, 4]), ("rewind", [102, 1, 39, 203]),
             (small, [1, 1, 1, 1]), ("rewind", [-1, -1, 0, -1]), (plan, [1, 64, 150, 1]), (small, [2, 1, 3, 1])]
    for p, new in steps:
        print(f"[paged run] {new}", flush=True)
        if p == "rewind":
            c.rewind(new)
            for x in o:
                x.rewind(new)
            continue
        ref = _extend(c, o[0], p, new)
        assert o[1].extend(new, p.max_tokens, p.max_new)["slots"].tolist() == ref["slots"].tolist()
        n = sum(new)
        for li in range(2):
            qkv = _values(g, (n, n_q + 2 * n_kv, D), torch.float16, dev, 0.2)
            q, k, v = qkv[:, :n_q], qkv[:, n_q:n_q + n_kv], qkv[:, n_q + n_kv:]
            qr = c.append(li, k, v, p, q=q, rotary=rot)
            q2, k2 = rot(q, k, p.positions[:n])
            assert torch.equal(qr, q2)
            o[li].append(_np(k2), _np(v), ref)
            _check_codes(c, o[li], li)
            want, bound = o[li].attend(_np(qr), ref, D ** -0.5)
            _check_attend(c.attend(li, qr, p), want, bound, torch.float16)
    k, v = c.read(1, 2)
    rk, rv = o[1].held(2, o[1].lens[2])
    assert np.array_equal(_np(k), rk) and np.array_equal(_np(v), rv)


@pytest.mark.parametrize("past,new,max_new", [([0], [700], None), ([5000, 20], [400, 300], None), ([0, 3000, 9, 800], [1, 1, 1, 1], None),
                                              ([3, 2000, 0], [60, 3, 500], None), ([0, 40, 5], [3, 4, 2], 4)])
def test_calls_with_fewer_tokens_than_the_step(dev, past, new, max_new):
    """The first tokens alone, with and without the rest of their row: their
    outputs, and nothing past them."""
    print(f"[attend] first tokens of {past} {new}", flush=True)
    c, o, plan, ref, q = _filled(dev, 32, 8, past, new, torch.float16, 8, max_new=max_new)
    want, bound = o.attend(_np(q), ref, D ** -0.5)
    total = sum(new)
    for n in sorted({1, 2, total // 3, total // 2, total - 1, total} - {0}):
        out = torch.full_like(q, 7.0)
        c.attend(0, q[:n], plan, out=out[:n])
        _check_attend(out[:n], want[:n], bound[:n], torch.float16)
        assert (out[n:] == 7.0).all()


def test_append_of_the_first_tokens_leaves_the_rest(dev):
    """Places of tokens that the call does not have keep their codes; those it
    has are coded as the oracle does with the step cut there."""
    for past, new, n in (([10, 100], [100, 60], 90), ([10, 100], [100, 60], 130), ([63, 0, 5], [2, 1, 2], 3)):
        print(f"[append] first {n} of {past} {new}", flush=True)
        g = torch.Generator(device=dev).manual_seed(9)
        rows = len(past)
        c, o = _pair(8, rows, 300, 12, dev)
        first, plan = c.new_plan(sum(past)), c.new_plan(sum(new), max_new=max(new))
        for p, lens, m in ((first, past, sum(past)), (plan, new, n)):
            ref = _extend(c, o, p, lens)
            k, v = (_values(g, (m, 8, D), torch.float16, dev) for _ in range(2))
            c.append(0, k, v, p)
            cut = [max(0, min(b, m) - a) for a, b in zip(ref["cu"], ref["cu"][1:])]
            ref["kv_len"] = [a + b for a, b in zip(ref["past"], cut)]
            o.append(_np(k), _np(v), ref)
        _check_codes(c, o)


def test_lengths_of_64_bits_do_not_wrap(dev):
    print("[tables] 64-bit lengths", flush=True)
    c, o = _pair(1, 3, 200, 12, dev, n_q=1)
    plan = c.new_plan(300)
    big = 2 ** 32
    c.extend(torch.tensor([70, big + 5, -big - 7], device=dev), plan)
    assert plan.rejected.tolist() == [0, 1, 1] and c.lens.tolist() == [70, 0, 0]
    c.rewind(torch.tensor([big + 1, -big, 0], device=dev))
    assert c.lens.tolist() == [70, 0, 0]


def test_pages_past_32_bit_offsets(dev):
    """A pool of 10 GB whose last pages are used: the same outputs and codes as
    in a small one."""
    print("[paged] 10 GB pool", flush=True)
    g = torch.Generator(device=dev).manual_seed(10)
    n_kv, past, new = 32, [700, 64], [1, 90]
    kv = [torch.randn((n, n_kv, D), generator=g, device=dev).half() for n in (sum(past), sum(past), sum(new), sum(new))]
    q = torch.randn((sum(new), 32, D), generator=g, device=dev).half()
    got = []
    for n_pages in (20, 20000):
        c = oi2.PagedKVCache(1, 32, n_kv, 2, 800, n_pages, device=dev)
        c.free.copy_(torch.arange(n_pages, dtype=torch.int32))          # the last pages first
        c.append(0, kv[0], kv[1], c.extend(past, c.new_plan(sum(past))))
        few = c.new_plan(sum(new), max_new=90)
        c.append(0, kv[2], kv[3], c.extend(new, few))
        assert int(c.block_table.max()) == n_pages - 1
        got.append((c.attend(0, q, few), *c.read(0, 0), *c.read(0, 1)))
        del c
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_query_that_is_not_finite_harms_no_other(dev, dtype, bad):
    print(f"[attend] query with {bad}", flush=True)
    for past, new in (([700, 90], [3, 1]), ([300, 5000], [150, 40])):
        c, o, plan, ref, q = _filled(dev, 32, 8, past, new, dtype, 11)
        y = c.attend(0, q, plan)
        t, h = sum(new) // 2, 9
        q[t, h, 5] = bad
        z = c.attend(0, q, plan)
        assert z[t, h].isnan().all()
        z[t, h] = y[t, h]
        assert torch.equal(z, y)
