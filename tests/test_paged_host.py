"""The paged cache's oracle on small examples, and what the product refuses.
CPU only: nothing here launches a kernel."""
import ctypes
import math

import numpy as np
import pytest
import torch

import oi2
from oi2 import _lib
from oracle import paged as P


def test_oracle_codes_are_torchs_casts():
    x = torch.cat([torch.linspace(-448, 448, 20001), torch.randn(5000) * 0.01, torch.tensor([0.0, 2 ** -10, 3 * 2 ** -10])])
    ref = x.to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(P.code(x.double().numpy(), 0), ref)
    assert np.array_equal(P.code(x.double().numpy() * 8, 3), ref)
    assert np.isnan(P.code([math.inf, -math.inf, math.nan, 449.0], 0)).all()


def test_oracle_exponents():
    for top, e in ((448.0, 0), (448.0001, 1), (449.0, 1), (1.75, -8), (1.7500001, -7), (1.0, -8), (0.0, -40), (2.0 ** -60, -40),
                   (1e38, 60), (math.inf, -40), (math.nan, -40), (896.0, 1)):
        assert P.exponent([top, -0.0]) == e, top
        if 0 < top < 1e20 and e > -40:
            assert top <= 448.0 * 2.0 ** e and top > 448.0 * 2.0 ** (e - 1)


def test_oracle_attention_of_a_hand_example():
    c = P.Cache(1, 10, 1, 1)
    plan = c.extend([2], 2, 2)
    k = np.zeros((2, 1, 128))
    v = np.zeros((2, 1, 128))
    k[1, 0, 0], v[0, 0, 5], v[1, 0, 5] = 1.0, 1.0, 3.0
    c.append(k, v, plan)
    q = np.zeros((2, 1, 128))
    q[:, 0, 0] = math.log(3.0)
    out, _ = c.attend(q, plan, 1.0)
    assert np.allclose(out[0, 0, 5], 1.0) and np.allclose(out[1, 0, 5], (1 + 3 * 3) / 4)


def test_rotary_frequencies():
    f, m = oi2.rotary_frequencies(8, 10000.0)
    assert np.allclose(f, [1.0, 0.1, 0.01, 0.001]) and m == 1.0
    f, _ = oi2.rotary_frequencies(8, 10000.0, {"type": "linear", "factor": 4.0})
    assert np.allclose(f, [0.25, 0.025, 0.0025, 0.00025])
    f, _ = oi2.rotary_frequencies(8, 10000.0, {"type": "ntk", "factor": 4.0})
    assert np.allclose(f[0], 1.0) and np.allclose(f[-1], 0.001 / 4.0)
    f, _ = oi2.rotary_frequencies(8, 10000.0, {"type": "wavelength", "factor": 4.0, "original_len": 2 * math.pi * 20,
                                               "low_factor": 1.0, "high_factor": 3.0})
    assert np.allclose(f, [1.0, 0.1 * 0.5 + 0.025 * 0.5, 0.0025, 0.00025])
    f, m = oi2.rotary_frequencies(64, 10000.0, {"type": "yarn", "factor": 16.0, "original_len": 4096, "beta_fast": 32.0,
                                                "beta_slow": 1.0})
    assert np.allclose(f[0], 1.0) and np.allclose(f[-1], 10000.0 ** (-62 / 64) / 16) and np.allclose(m, 0.1 * math.log(16) + 1)


@pytest.mark.parametrize("bad", [
    {"type": "other"}, {"factor": 2.0}, {"type": "linear"}, {"type": "linear", "factor": 0.0},
    {"type": "linear", "factor": math.inf}, {"type": "linear", "factor": 2.0, "more": 1.0},
    {"type": "wavelength", "factor": 8.0, "original_len": 8192, "low_factor": 4.0, "high_factor": 4.0},
])
def test_rotary_scalings_refused(bad):
    with pytest.raises(ValueError):
        oi2.rotary_frequencies(64, 10000.0, bad)


def test_theta_refused():
    for theta in (1.0, 0.0, -5.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            oi2.rotary_frequencies(64, theta)


@pytest.mark.parametrize("kw", [
    {"n_kv": 3}, {"n_kv": 0}, {"n_q": 16, "n_kv": 1}, {"n_seqs": 0}, {"n_seqs": 2049}, {"max_len": 0}, {"max_len": 2 ** 31},
    {"n_pages": 0}, {"n_pages": 2 ** 25}, {"n_layers": -1}, {},
])
def test_cache_sizes_refused(kw):
    """The empty one: tables on the CPU are refused too."""
    args = dict(n_layers=1, n_q=32, n_kv=8, n_seqs=4, max_len=100, n_pages=10)
    with pytest.raises(ValueError):
        oi2.PagedKVCache(**{**args, **kw}, device="cpu")


def _structs(**kw):
    c = dict(n_q=32, n_kv=8, n_seqs=4, max_len=100, n_pages=10, n_layers=2, block_table=64, lens=64, free_pages=64, n_free=64,
             pages=64, scales=64)
    p = dict(max_tokens=16, max_new=4, cu=64, positions=64, slots=64, kv_len=64, rejected=64, work=64)
    r = dict(head_dim=128, rotary_dim=128, interleaved=0, magnitude=1.0, freq=64)
    h = dict(k=_lib.Heads(64, 8, 1024, 128), v=_lib.Heads(64, 8, 1024, 128), q=_lib.Heads(64, 32, 4096, 128))
    for k, v in kw.items():
        for d in (c, p, r):
            if k in d:
                d[k] = v
    return _lib.Paged(**c), _lib.PagePlan(**p), _lib.Rotary(**r), {**h, **{k: v for k, v in kw.items() if k in h}}


REFUSED = [
    ("extend", dict(n_kv=5), b"kv heads"), ("extend", dict(n_seqs=3000), b"rows"), ("extend", dict(n_pages=2 ** 25), b"pages"),
    ("extend", dict(max_tokens=0), b"plan of 0"), ("extend", dict(max_new=0), b"plan of"), ("extend", dict(block_table=None), b"null"),
    ("extend", dict(cu=None), b"null"), ("extend", dict(work=None), b"null"), ("extend", dict(work=68), b"aligned"),
    ("rewind", dict(lens=None), b"null"), ("rewind", dict(n_q=7), b"heads"),
    ("append", dict(pages=None), b"pages"), ("append", dict(pages=72), b"aligned"), ("append", dict(scales=68), b"scales"),
    ("append", dict(layer=2), b"layer"), ("append", dict(layer=-1), b"layer"), ("append", dict(dtype=0), b"dtype"),
    ("append", dict(n=17), b"17 tokens"), ("append", dict(n=-1), b"-1 tokens"), ("append", dict(k=_lib.Heads(64, 4, 512, 128)), b"heads"),
    ("append", dict(v=_lib.Heads(65, 8, 1024, 128)), b"aligned"), ("append", dict(k=_lib.Heads(None, 8, 1024, 128)), b"null"),
    ("append", dict(rotary_dim=130), b"rotary_dim"), ("append", dict(rotary_dim=3), b"rotary_dim"), ("append", dict(freq=None), b"null"),
    ("append", dict(head_dim=64, rotary_dim=64), b"head_dim"), ("append", dict(q=_lib.Heads(None, 32, 4096, 128)), b"q and its"),
    ("attend", dict(dtype=7), b"dtype"), ("attend", dict(n=17), b"tokens"), ("attend", dict(q=_lib.Heads(64, 8, 1024, 128)), b"query heads"),
    ("attend", dict(scale=math.nan), b"finite"), ("attend", dict(scale=math.inf), b"finite"), ("attend", dict(out=None), b"out"),
    ("attend", dict(out=72), b"out"), ("attend", dict(layer=2), b"layer"), ("attend", dict(ws=0, max_len=5000), b"workspace"),
    ("attend", dict(q=_lib.Heads(65, 32, 4096, 128)), b"aligned"),
    ("rotary", dict(dtype=0), b"dtype"), ("rotary", dict(head_dim=258), b"head_dim"), ("rotary", dict(n=-1), b"tokens"),
    ("rotary", dict(rotary_dim=0), b"rotary_dim"), ("rotary", dict(positions_arg=None), b"positions"),
    ("rotary", dict(q=_lib.Heads(64, -1, 1, 1)), b"heads"), ("rotary", dict(q=_lib.Heads(65, 32, 4096, 128)), b"aligned"),
    ("rotary", dict(n=2 ** 31 - 1), b"too many"),
]


@pytest.mark.parametrize("call,kw,says", REFUSED)
def test_refusals_of_the_c_abi(call, kw, says):
    """Checked on the host before anything is launched; addresses here are
    numbers that nothing reads."""
    lib = oi2.load_library()
    c, p, r, h = _structs(**kw)
    ref = ctypes.byref
    n, layer, dtype = kw.get("n", 4), kw.get("layer", 0), kw.get("dtype", _lib.DTYPE_F16)
    if call == "extend":
        rc = lib.oi2_page_extend(ref(c), ref(p), 64, None)
    elif call == "rewind":
        rc = lib.oi2_page_rewind(ref(c), kw.get("lens", 64), None)
    elif call == "append":
        rc = lib.oi2_kv_append(ref(c), ref(p), layer, dtype, n, ref(h["k"]), ref(h["v"]), ref(r), ref(h["q"]), 64, None)
    elif call == "attend":
        rc = lib.oi2_kv_attend(ref(c), ref(p), layer, dtype, n, ref(h["q"]), kw.get("scale", 0.1), kw.get("out", 64), 64,
                               kw.get("ws", 1 << 40), None)
    else:
        rc = lib.oi2_rotary_apply(ref(r), dtype, n, kw.get("positions_arg", 64), ref(h["q"]), 64, ref(h["k"]), 64, None)
    assert rc == 1
    assert says in lib.oi2_last_error(), lib.oi2_last_error()


def test_null_structs_are_refused():
    lib = oi2.load_library()
    c, p, r, h = _structs()
    ref = ctypes.byref
    assert lib.oi2_page_extend(None, ref(p), 64, None) == 1
    assert lib.oi2_page_extend(ref(c), None, 64, None) == 1
    assert lib.oi2_page_extend(ref(c), ref(p), None, None) == 1
    assert lib.oi2_kv_append(ref(c), ref(p), 0, 2, 4, None, ref(h["v"]), None, None, None, None) == 1
    assert lib.oi2_kv_append(ref(c), ref(p), 0, 2, 4, ref(h["k"]), ref(h["v"]), None, ref(h["q"]), 64, None) == 1
    assert lib.oi2_kv_attend(ref(c), ref(p), 0, 2, 4, None, 0.1, 64, 64, 1 << 40, None) == 1
    assert lib.oi2_rotary_apply(None, 2, 4, 64, ref(h["q"]), 64, ref(h["k"]), 64, None) == 1
    assert lib.oi2_rotary_apply(ref(r), 2, 4, 64, None, 64, ref(h["k"]), 64, None) == 1
    assert lib.oi2_page_plan_bytes(None, 4, 4) == 0 and lib.oi2_page_plan_bytes(ref(c), 0, 4) == 0
    assert lib.oi2_kv_attend_workspace_bytes(ref(c), 4, 0) == 0
    assert lib.oi2_kv_append(ref(c), ref(p), 0, 2, 0, ref(h["k"]), ref(h["v"]), None, None, None, None) == 0    # no token: nothing to do


@pytest.mark.parametrize("kw,says", [
    (dict(n_kv=4), b"4 kv heads on a cache of 32 and 8"), (dict(n_q=16), b"16 query"), (dict(layer=2), b"layer"), (dict(pages=None), b"pages"),
    (dict(cu=None), b"null"), (dict(head_dim=64, rotary_dim=64), b"head_dim"), (dict(n=17), b"17 tokens"), (dict(n=-1), b"-1 tokens"),
    (dict(x=None), b"x must"), (dict(x=72), b"x must"), (dict(wq=None), b"null weight"), (dict(wo=72), b"weights must"),
    (dict(norm_w=None), b"norm"), (dict(out=None), b"output"), (dict(ws=1000), b"workspace"),
])
def test_layer_refusals_of_the_c_abi(kw, says):
    lib = oi2.load_library()
    c, p, r, _ = _structs(**{k: v for k, v in kw.items() if k not in ("n_q", "n_kv")})
    w = dict(wq=64, wk=64, wv=64, wo=64, n_q=32, n_kv=8, norm_w=64)
    w = _lib.Attn(**{**w, **{k: v for k, v in kw.items() if k in w}})
    ref = ctypes.byref

    def call(n):
        return lib.oi2_attn_forward_paged(kw.get("x", 64), n, ref(w), 1e-5, ref(r), ref(c), ref(p), kw.get("layer", 0),
                                          kw.get("out", 64), None, 64, kw.get("ws", 1 << 40), None)
    assert call(kw.get("n", 4)) == 1
    assert says in lib.oi2_last_error(), lib.oi2_last_error()


def test_layer_null_structs_and_no_tokens():
    lib = oi2.load_library()
    c, p, r, _ = _structs()
    w = _lib.Attn(wq=64, wk=64, wv=64, wo=64, n_q=32, n_kv=8, norm_w=64)
    ref = ctypes.byref
    for drop in range(4):
        a = [None if i == drop else ref(x) for i, x in enumerate((w, r, c, p))]
        assert lib.oi2_attn_forward_paged(64, 4, a[0], 1e-5, a[1], a[2], a[3], 0, 64, None, 64, 1 << 40, None) == 1
    assert lib.oi2_attn_forward_paged(64, 0, ref(w), 1e-5, ref(r), ref(c), ref(p), 0, 64, None, 64, 1 << 40, None) == 0
    assert lib.oi2_attn_paged_workspace_bytes(None, 4, 4, 4) == 0
    assert lib.oi2_attn_paged_workspace_bytes(ref(c), 4, 4, 5) == 0 and lib.oi2_attn_paged_workspace_bytes(ref(c), 4, 4, 0) == 0
