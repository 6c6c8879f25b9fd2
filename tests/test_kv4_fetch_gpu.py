"""Positions of a 4-bit cache read back into outputs that are slices of one
buffer, bit for bit against the float64 oracle.
"""
import itertools

import pytest
import torch

from tests.test_gpu_paged import dev  # noqa: F401
from tests.test_kv4_gpu import _held

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
