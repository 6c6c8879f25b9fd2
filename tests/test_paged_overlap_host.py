"""Outputs of the rotary and paged operators that share memory with what other
workgroups read: refused on the host.  Addresses here are numbers that nothing
reads; calls that would launch are not made."""
import ctypes

import pytest
import torch

import oi2
from oi2 import _lib

N, D = 4, 128
AT = 1 << 20                       # an address; a token of 8 heads has 2048 bytes


def _heads(at, heads, token=None, head=D):
    return _lib.Heads(at, heads, heads * D if token is None else token, head)


def _cache():
    c = _lib.Paged(n_q=8, n_kv=8, n_seqs=4, max_len=100, n_pages=10, n_layers=1, block_table=64, lens=64, free_pages=64, n_free=64,
                   pages=64, scales=64)
    p = _lib.PagePlan(max_tokens=16, max_new=4, cu=64, positions=64, slots=64, kv_len=64, rejected=64, work=64)
    r = _lib.Rotary(head_dim=D, rotary_dim=D, interleaved=0, magnitude=1.0, freq=64)
    return c, p, r


SIZE = N * 8 * D * 2               # bytes of q, k, or an output
FAR = [AT + 10 * SIZE * i for i in range(1, 6)]
# q, q_out, k, k_out: what clashes
ROTARY = [
    ("q_out behind q's start", AT, AT + 2, FAR[0], FAR[1]), ("q_out before q's end", AT, AT + SIZE - 16, FAR[0], FAR[1]),
    ("q_out's end in q", AT, AT - SIZE + 16, FAR[0], FAR[1]), ("q_out is k", AT, FAR[0], FAR[0], FAR[1]),
    ("k_out is q", AT, FAR[0], FAR[1], AT), ("k_out in k", AT, AT, FAR[0], FAR[0] + 256), ("q_out is k_out", AT, FAR[0], FAR[1], FAR[0]),
    ("q_out meets k_out", AT, FAR[0], FAR[1], FAR[0] + SIZE - 2), ("each the other's", AT, FAR[0], FAR[0], AT),
]


@pytest.mark.parametrize("what,q,qo,k,ko", ROTARY)
def test_rotary(what, q, qo, k, ko):
    lib = oi2.load_library()
    _, _, r = _cache()
    ref = ctypes.byref
    assert lib.oi2_rotary_apply(ref(r), _lib.DTYPE_F16, N, 64, ref(_heads(q, 8)), qo, ref(_heads(k, 8)), ko, None) == 1
    assert b"shares memory" in lib.oi2_last_error()


@pytest.mark.parametrize("what,q,qo,k,v", [
    ("in q", _heads(AT, 8), AT + 16, _heads(FAR[0], 8), _heads(FAR[1], 8)), ("is k", _heads(AT, 8), FAR[0], _heads(FAR[0], 8), _heads(FAR[1], 8)),
    ("in v", _heads(AT, 8), FAR[1] + SIZE - 2, _heads(FAR[0], 8), _heads(FAR[1], 8)),
    ("of a fused row", _heads(AT, 8, 24 * D), AT, _heads(AT + 16 * D, 8, 24 * D), _heads(AT + 32 * D, 8, 24 * D)),
    ("heads first", _heads(AT, 8, D, N * D), AT, _heads(FAR[0], 8), _heads(FAR[1], 8)),
    ("backwards", _heads(AT + SIZE, 8, -8 * D), AT + SIZE - 16 * D, _heads(FAR[0], 8), _heads(FAR[1], 8)),
])
def test_append(what, q, qo, k, v):
    lib = oi2.load_library()
    c, p, r = _cache()
    ref = ctypes.byref
    assert lib.oi2_kv_append(ref(c), ref(p), 0, _lib.DTYPE_BF16, N, ref(k), ref(v), ref(r), ref(q), qo, None) == 1
    assert b"shares memory" in lib.oi2_last_error()


@pytest.mark.parametrize("q,out", [(_heads(AT, 8), AT + 16), (_heads(AT, 8), AT - SIZE + 16), (_heads(AT, 8, 24 * D), AT),
                                   (_heads(AT, 8, D, N * D), AT)])
def test_attend(q, out):
    lib = oi2.load_library()
    c, p, _ = _cache()
    ref = ctypes.byref
    assert lib.oi2_kv_attend(ref(c), ref(p), 0, _lib.DTYPE_F16, N, ref(q), 0.1, out, 1 << 40, 1 << 40, None) == 1
    assert b"shares memory" in lib.oi2_last_error()


def test_spans():
    x = torch.zeros(6, 4, 8)
    assert _lib.overlap(x, x) and _lib.overlap(x[:, 1:3], x[2]) and not _lib.overlap(x[:3], x[3:])
    assert not _lib.overlap(x[:0], x) and not _lib.overlap(x, torch.zeros(3)) and _lib.overlap(x[2:5], x[4:])
