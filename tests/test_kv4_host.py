"""The paged 4-bit cache without a GPU: the oracle's codes, the C ABI's refusals,
and the layout of a dword that the header gives."""
import ctypes
import math

import numpy as np
import pytest
import torch

import oi2
from oi2 import _lib
from oracle import paged4 as P

AT = 1 << 20


def _structs(**kw):
    c = dict(n_q=32, n_kv=8, n_seqs=4, max_len=1000, n_pages=100, n_layers=2, block_table=64, lens=64, free_pages=64, n_free=64, pages=64,
             scales=None)
    p = dict(max_tokens=16, max_new=4, cu=64, positions=64, slots=64, kv_len=64, rejected=64, work=64)
    r = dict(head_dim=128, rotary_dim=128, interleaved=0, magnitude=1.0, freq=64)
    h = dict(q=_lib.Heads(AT, 32, 4096, 128), k=_lib.Heads(AT << 1, 8, 1024, 128), v=_lib.Heads(AT << 2, 8, 1024, 128))
    for d in (c, p, r, h):
        d.update({k: v for k, v in kw.items() if k in d})
    return _lib.Paged(**c), _lib.PagePlan(**p), _lib.Rotary(**r), h


REFUSED = [
    ("append", dict(pages=None), b"pages"), ("append", dict(pages=72), b"aligned"), ("append", dict(layer=2), b"layer"),
    ("append", dict(layer=-1), b"layer"), ("append", dict(dtype=0), b"dtype"), ("append", dict(n=17), b"17 tokens"),
    ("append", dict(n=-1), b"-1 tokens"), ("append", dict(k=_lib.Heads(64, 4, 512, 128)), b"heads"),
    ("append", dict(v=_lib.Heads(65, 8, 1024, 128)), b"aligned"), ("append", dict(rotary_dim=130), b"rotary_dim"),
    ("append", dict(head_dim=64, rotary_dim=64), b"head_dim"), ("append", dict(n_seqs=3000), b"rows"), ("append", dict(slots=None), b"null"),
    ("append", dict(q=_lib.Heads(AT + 16, 32, 4096, 128)), b"shares memory"), ("append", dict(k=_lib.Heads(AT + 64, 8, 1024, 128)), b"shares memory"),
    ("attend", dict(dtype=7), b"dtype"), ("attend", dict(n=17), b"tokens"), ("attend", dict(q=_lib.Heads(64, 8, 1024, 128)), b"query heads"),
    ("attend", dict(scale=math.nan), b"finite"), ("attend", dict(scale=-math.inf), b"finite"), ("attend", dict(out=None), b"out"),
    ("attend", dict(out=72), b"out"), ("attend", dict(layer=2), b"layer"), ("attend", dict(ws=0, max_len=5000), b"workspace"),
    ("attend", dict(pages=None), b"pages"), ("attend", dict(out=AT + 64), b"shares memory"),
    ("fetch", dict(dtype=7), b"dtype"), ("fetch", dict(n=-1), b"tokens"), ("fetch", dict(count=None), b"null"), ("fetch", dict(cu_out=None), b"null"),
    ("fetch", dict(layer=-1), b"layer"), ("fetch", dict(pages=None), b"pages"), ("fetch", dict(k=_lib.Heads(None, 8, 1024, 128)), b"non-null"),
    ("fetch", dict(k=_lib.Heads(AT, 4, 1024, 128)), b"heads"), ("fetch", dict(v=_lib.Heads(AT + 1, 8, 1024, 128)), b"aligned"),
    # a cache of 8 bits
    ("append", dict(scales=64), b"scales"), ("attend", dict(scales=64), b"scales"), ("fetch", dict(scales=64), b"scales"),
    # cu where the counts are, or where they end
    ("fetch", dict(count=AT, cu_out=AT), b"shares memory"), ("fetch", dict(count=AT, cu_out=AT + 12), b"shares memory"),
    ("fetch", dict(count=AT, cu_out=AT - 16), b"shares memory"), ("fetch", dict(lens=AT, cu_out=AT + 4), b"shares memory"),
    # an output's values in one place, or backwards
    ("fetch", dict(k=_lib.Heads(AT, 8, 0, 128)), b"share memory"), ("fetch", dict(k=_lib.Heads(AT, 8, 1024, 64)), b"share memory"),
    ("fetch", dict(k=_lib.Heads(AT, 8, 1023, 128)), b"share memory"), ("fetch", dict(v=_lib.Heads(AT, 8, -1024, 128)), b"share memory"),
    ("fetch", dict(k=_lib.Heads(AT, 8, 128, 511)), b"share memory"),
    # k and v
    ("fetch", dict(k=_lib.Heads(AT, 8, 1024, 128), v=_lib.Heads(AT, 8, 1024, 128)), b"share memory"),
    ("fetch", dict(k=_lib.Heads(AT, 8, 1024, 128), v=_lib.Heads(AT + 8192 - 256, 8, 1024, 128)), b"share memory"),
    ("fetch", dict(k=_lib.Heads(AT, 8, 2048, 128), v=_lib.Heads(AT + 1024, 8, 2048, 128)), b"share memory"),
    ("fetch", dict(k=_lib.Heads(AT, 8, 2048, 128), v=_lib.Heads(AT + 2048, 8, 2048, 256)), b"share memory"),
]


@pytest.mark.parametrize("call,kw,says", REFUSED)
def test_refusals_of_the_c_abi(call, kw, says):
    """Checked on the host before anything is launched; addresses here are
    numbers that nothing reads."""
    lib = oi2.load_library()
    c, p, r, h = _structs(**kw)
    ref = ctypes.byref
    n, layer, dtype = kw.get("n", 4), kw.get("layer", 0), kw.get("dtype", _lib.DTYPE_F16)
    if call == "append":
        rc = lib.oi2_kv4_append(ref(c), ref(p), layer, dtype, n, ref(h["k"]), ref(h["v"]), ref(r), ref(h["q"]), AT, None)
    elif call == "attend":
        rc = lib.oi2_kv4_attend(ref(c), ref(p), layer, dtype, n, ref(h["q"]), kw.get("scale", 0.1), kw.get("out", 1 << 30), 64,
                                kw.get("ws", 1 << 40), None)
    else:
        rc = lib.oi2_kv4_fetch(ref(c), layer, None, kw.get("count", 64), dtype, n, ref(h["k"]), ref(h["v"]), kw.get("cu_out", 64), None)
    assert rc == 1
    assert says in lib.oi2_last_error(), lib.oi2_last_error()


def test_null_structs_and_no_tokens():
    lib = oi2.load_library()
    c, p, r, h = _structs()
    ref = ctypes.byref
    assert lib.oi2_kv4_append(None, ref(p), 0, 2, 4, ref(h["k"]), ref(h["v"]), None, None, None, None) == 1
    assert lib.oi2_kv4_append(ref(c), None, 0, 2, 4, ref(h["k"]), ref(h["v"]), None, None, None, None) == 1
    assert lib.oi2_kv4_append(ref(c), ref(p), 0, 2, 4, None, ref(h["v"]), None, None, None, None) == 1
    assert lib.oi2_kv4_append(ref(c), ref(p), 0, 2, 4, ref(h["k"]), ref(h["v"]), None, ref(h["q"]), AT, None) == 1
    assert lib.oi2_kv4_append(ref(c), ref(p), 0, 2, 0, ref(h["k"]), ref(h["v"]), None, None, None, None) == 0
    assert lib.oi2_kv4_attend(ref(c), ref(p), 0, 2, 4, None, 0.1, 64, 64, 1 << 40, None) == 1
    assert lib.oi2_kv4_attend(ref(c), None, 0, 2, 4, ref(h["q"]), 0.1, 64, 64, 1 << 40, None) == 1
    assert lib.oi2_kv4_attend(ref(c), ref(p), 0, 2, 0, ref(h["q"]), 0.1, 64, 64, 1 << 40, None) == 0
    assert lib.oi2_kv4_fetch(None, 0, None, 64, 2, 4, ref(h["k"]), ref(h["v"]), 64, None) == 1
    assert lib.oi2_kv4_fetch(ref(c), 0, None, 64, 2, 4, None, ref(h["v"]), 64, None) == 1
    w = _lib.Attn(wq=64, wk=64, wv=64, wo=64, n_q=32, n_kv=8, norm_w=64)
    for drop in range(4):
        a = [None if i == drop else ref(x) for i, x in enumerate((w, r, c, p))]
        assert lib.oi2_kv4_attn_forward(64, 4, a[0], 1e-5, a[1], a[2], a[3], 0, 64, None, 64, 1 << 40, None) == 1
    assert lib.oi2_kv4_attn_forward(64, 4, ref(w), 1e-5, ref(r), ref(c), ref(p), 2, 64, None, 64, 1 << 40, None) == 1
    assert b"layer" in lib.oi2_last_error()
    assert lib.oi2_kv4_attn_forward(64, 0, ref(w), 1e-5, ref(r), ref(c), ref(p), 0, 64, None, 64, 1 << 40, None) == 0


def test_bits_are_4_or_8():
    for bits in (0, 2, 16, None, "4"):
        with pytest.raises(ValueError):
            oi2.PagedKVCache(1, 8, 8, 1, 64, 1, bits=bits)


def test_oracle_codes():
    """Scales and codes by hand: a full range, ties, the scale's rounding, the
    smallest and largest, groups that are not finite."""
    x = np.zeros((6, 128))
    x[0, :15] = np.arange(-7, 8)                   # scale 1
    x[0, 32:40] = [7, 0.5, 1.5, -2.5, 3.5, 0.25, -0.75, 6.5]
    x[1, 0] = 7 * (1 + 2.0 ** -8)                  # a tie of the scale's 8 bits: to even
    x[1, 32] = 7 * (1 + 3 * 2.0 ** -8)
    x[1, 64] = 2.0 ** -24
    x[1, 65] = -(2.0 ** -26)
    x[2, 0], x[2, 1] = 1e30, -1.0
    x[3, 5], x[3, 40], x[3, 70] = np.nan, np.inf, -np.inf
    n, s = P.code(x)
    assert s[0, 0] == 1 and n[0, 0, :15].tolist() == list(range(-7, 8))
    assert n[0, 1, :8].tolist() == [7, 0, 2, -2, 4, 0, -1, 6]
    assert s[1, 0] == 1 and s[1, 1] == 1 + 2.0 ** -6
    assert s[1, 2] == 2.0 ** -24 and n[1, 2, 0] == 1 and n[1, 2, 1] == 0
    assert s[2, 0] == 9344 and n[2, 0, 0] == 7 and n[2, 0, 1] == 0
    assert np.isnan(s[3]).tolist() == [True, True, True, False] and not n[3].any()
    assert not s[4].any() and not n[4].any()
    # exact in fp16, whatever the values
    g = np.random.default_rng(1)
    y = (g.standard_normal((300, 128)) * np.exp2(g.integers(-24, 16, (300, 1)))).clip(-65504, 65504).astype(np.float16).astype(np.float64)
    n, s = P.code(y)
    z = n * s[..., None]
    assert np.array_equal(z.astype(np.float16).astype(np.float64), z)
    # off by half the scale: 7 of a scale that was rounded down miss the largest
    # value by 7 times what it lost, 2^-8 of it, or 2^-25 where it is small
    err = np.abs(z.reshape(300, 128) - y).reshape(300, 4, 32)
    assert (err <= np.maximum(0.5 * s, 7 * 2.0 ** -25)[..., None]).all()


def test_dword_of_the_header():
    """The header's places of magnitudes and signs are 32 different bits."""
    e = np.arange(4)
    bits = np.concatenate([8 * e + b for b in range(3)] + [8 * e + 4 + b for b in range(3)] + [8 * e + 7, (8 * e + 11) % 32])
    assert sorted(bits.tolist()) == list(range(32))
    k = [1024 * (p // 4 % 4) + 256 * (u // 4) + 16 * (4 * (p // 16) + p % 4) + 4 * (u % 4) for p in range(64) for u in range(16)]
    v = [1024 * (p // 4 % 4) + 256 * (p // 16) + 16 * u + 4 * (p % 4) for p in range(64) for u in range(16)]
    ks = [8 * (16 * c + 4 * (p // 16) + p % 4) + 2 * (p // 4 % 4) for p in range(64) for c in range(4)]
    assert sorted(k) == sorted(v) == list(range(0, 4096, 4)) and sorted(ks) == list(range(0, 512, 2))
