"""Where fetch's outputs may lie, without a GPU: the check of the C entry against
every value's place counted one by one.  What it lets through reaches the check
behind it, which these calls fail, so that nothing is launched."""
import ctypes
import itertools
import random

import pytest

import oi2
from oi2 import _lib

AT = 1 << 24


def _fetch(k, v, tokens, heads, dtype=_lib.DTYPE_F16):
    """None where k and v are taken, else what is said; k, v: (address, token
    stride, head stride)."""
    lib = oi2.load_library()
    c = _lib.Paged(n_q=heads, n_kv=heads, n_seqs=4, max_len=1000, n_pages=100, n_layers=1, block_table=64, lens=64, free_pages=64,
                   n_free=64, pages=64, scales=None)
    hk, hv = (_lib.Heads(x[0], heads, x[1], x[2]) for x in (k, v))
    ref = ctypes.byref
    assert lib.oi2_kv4_fetch(ref(c), 0, None, 1024, dtype, tokens, ref(hk), ref(hv), 1024, None) == 1   # cu where the counts are
    said = lib.oi2_last_error().decode()
    return None if "cu shares memory with what is read" in said else said


def _places(x, tokens, heads, size):
    return [x[0] // size + t * x[1] + h * x[2] for t in range(tokens) for h in range(heads)]


def _meet(places):
    places = sorted(places)
    return any(b - a < 128 for a, b in zip(places, places[1:]))


@pytest.mark.parametrize("tokens", [1, 2, 37])
@pytest.mark.parametrize("heads", [1, 3, 8])
@pytest.mark.parametrize("dtype,size", [(_lib.DTYPE_F16, 2), (_lib.DTYPE_F32, 4)])
def test_layouts_of_one_buffer(tokens, heads, dtype, size):
    """k and v in one buffer, whichever dimension comes first, with their places
    exchanged, and with a gap behind the values."""
    for gap in (0, 8, 1):
        row = 128 + gap
        for order in itertools.permutations(["kv", "t", "h"]):
            n = {"kv": 2, "t": tokens, "h": heads}
            at, stride = row, {}
            for d in reversed(order):
                stride[d] = at
                at *= n[d]
            k, v = ((AT + i * stride["kv"] * size, stride["t"], stride["h"]) for i in range(2))
            assert _fetch(k, v, tokens, heads, dtype) is None, order
            assert _fetch(v, k, tokens, heads, dtype) is None, order


def test_against_every_place():
    """Strides and distances at random: taken where no two values meet, and k and
    v within one another's span lie alike; refused where any two meet."""
    rng = random.Random(3)
    seen = {True: 0, False: 0}
    for _ in range(6000):
        tokens, heads = rng.randint(1, 6), rng.randint(1, 5)
        unit = rng.choice([64, 127, 128, 128, 129, 130])
        st, sh = unit * rng.randint(0, 12), unit * rng.randint(0, 12)
        k, v = ((AT + 2 * (unit * rng.randint(0, 24) + rng.choice([0, 0, 0, 1, -1])), st, sh) for _ in range(2))
        meet = _meet(_places(k, tokens, heads, 2) + _places(v, tokens, heads, 2))
        assert (_fetch(k, v, tokens, heads) is not None) == meet, (k, v, tokens, heads)
        seen[meet] += 1
    assert min(seen.values()) > 500


def test_strides_of_their_own():
    """k and v laid out each in its way: taken behind one another, refused where
    their spans meet."""
    k, v = (AT, 1024, 128), (AT + 2 * 8 * 1024, 128, 8 * 128)
    assert _fetch(k, v, 8, 8) is None and _fetch(v, k, 8, 8) is None
    assert "share memory" in _fetch(k, (v[0] - 2, *v[1:]), 8, 8)
    # one token, one head: the stride of tokens, of heads, says nothing
    assert _fetch((AT, 5, 256), (AT + 256, 9, 256), 1, 8) is None
    assert _fetch((AT, 256, 5), (AT + 256, 256, 9), 8, 1) is None
    assert "share memory" in _fetch((AT, 5, 256), (AT + 254, 9, 256), 1, 8)
    assert "share memory" in _fetch((AT, 256, 128), (AT, 256, 128), 1, 1)


READ = [("first", 4), ("count", 4), ("lens", 4), ("block_table", 4 * 16), ("cu", 5)]


@pytest.mark.parametrize("what,ints", READ)
@pytest.mark.parametrize("which", ["k", "v"])
def test_outputs_over_what_is_read(which, what, ints):
    """k and v are refused where they share memory with counts, lengths, table or
    sums, at either end; so are sums where the table lies.  4 rows of 16 pages."""
    lib, ref = oi2.load_library(), ctypes.byref
    tokens, heads, size = 8, 2, 8 * 2 * 128 * 2
    for at in (AT, AT + size - 4, AT - 4 * ints + 4, AT + 512):
        where = dict(first=1024, count=2048, lens=3072, block_table=4096, cu=8192)
        where[what] = at
        c = _lib.Paged(n_q=heads, n_kv=heads, n_seqs=4, max_len=1000, n_pages=1, n_layers=1, block_table=where["block_table"],
                       lens=where["lens"], free_pages=64, n_free=64, pages=1 << 20, scales=None)
        other = _lib.Heads(AT << 1, heads, 256, 128)
        mine = _lib.Heads(AT, heads, 256, 128)
        k, v = (mine, other) if which == "k" else (other, mine)
        rc = lib.oi2_kv4_fetch(ref(c), 0, where["first"], where["count"], _lib.DTYPE_F16, tokens, ref(k), ref(v), where["cu"], None)
        assert rc == 1 and b"shares memory with what is read" in lib.oi2_last_error(), (at, lib.oi2_last_error())


def test_outputs_over_the_pages():
    lib, ref = oi2.load_library(), ctypes.byref
    c = _lib.Paged(n_q=2, n_kv=2, n_seqs=4, max_len=1000, n_pages=3, n_layers=2, block_table=4096, lens=3072, free_pages=64, n_free=64,
                   pages=1 << 20, scales=None)
    end = (1 << 20) + 2 * 3 * 2 * 9216
    k, v = _lib.Heads(AT, 2, 256, 128), _lib.Heads(AT << 1, 2, 256, 128)
    for bad in ((1 << 20) - 4096 + 16, end - 16):
        x = _lib.Heads(bad, 2, 256, 128)
        for a, b in ((x, v), (k, x)):
            assert lib.oi2_kv4_fetch(ref(c), 0, None, 2048, _lib.DTYPE_F16, 8, ref(a), ref(b), 8192, None) == 1
            assert b"shares memory with what is read" in lib.oi2_last_error()
    for cu in (end - 4, 4096 - 4, 4096 + 4 * 4 * 16 - 4):
        assert lib.oi2_kv4_fetch(ref(c), 0, None, 2048, _lib.DTYPE_F16, 8, ref(k), ref(v), cu, None) == 1
        assert b"cu shares memory with what is read" in lib.oi2_last_error()
