"""What the packed selection of a cold set refuses, on the host before any launch:
addresses here are numbers that nothing reads."""
import ctypes

import pytest

import oi2
from oi2 import _lib


def _call(**kw):
    lib = oi2.load_library()
    c = _lib.Paged(**{**dict(n_q=32, n_kv=8, n_seqs=4, max_len=100, n_pages=10, n_layers=0, block_table=64, lens=64, free_pages=64,
                             n_free=64, pages=None, scales=None), **kw.get("cache", {})})
    p = _lib.PagePlan(**{**dict(max_tokens=16, max_new=4, cu=64, positions=64, slots=64, kv_len=64, rejected=64, work=64),
                         **kw.get("plan", {})})
    pred = _lib.Predictor(1024, kw.get("rank", 64), _lib.DTYPE_F32, 64, 64, 64)
    ref = ctypes.byref
    rc = lib.oi2_predict_select_packed(kw.get("x", 64), kw.get("n", 4), ref(c), ref(p), kw.get("norm", 64), 1e-5, ref(pred), 0.0, 64,
                                       kw.get("slots", 64), 64, 64, kw.get("ws", 64), kw.get("bytes", 1 << 30), None)
    return rc, lib.oi2_last_error()


@pytest.mark.parametrize("kw,says", [
    (dict(x=None), b"x must"), (dict(x=72), b"x must"), (dict(n=0), b"0 tokens"), (dict(n=17), b"17 tokens in a plan of 16"),
    (dict(cache=dict(n_seqs=0)), b"rows"), (dict(cache=dict(lens=None)), b"null cache table"), (dict(plan=dict(cu=None)), b"null plan"),
    (dict(norm=72), b"norm_w"), (dict(slots=None), b"selection outputs"), (dict(ws=None), b"workspace"), (dict(bytes=64), b"workspace"),
    (dict(ws=72), b"workspace"), (dict(rank=3), b"rank"),
])
def test_refusals(kw, says):
    rc, error = _call(**kw)
    assert rc == 1 and says in error, error


def test_workspace_sizes():
    lib = oi2.load_library()
    pred = _lib.Predictor(1024, 64, _lib.DTYPE_F32, 64, 64, 64)
    plain = lib.oi2_predict_workspace_bytes(ctypes.byref(pred))
    for n in (1, 7, 2048):
        assert lib.oi2_predict_packed_workspace_bytes(ctypes.byref(pred), n) == plain + 8 * n
    for n in (-1, 0, 2049):
        assert lib.oi2_predict_packed_workspace_bytes(ctypes.byref(pred), n) == 0
