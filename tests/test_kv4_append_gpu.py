"""Appends of 4 bits so long that a workgroup takes several kv heads, whose
turns its threads share: the same q and pages as rotating first, in a call of its
own, and then appending what is rotated (a workgroup a head, by itself)."""
import pytest
import torch

import oi2
from tests.test_gpu_paged import SCALINGS, _values, dev  # noqa: F401

pytestmark = pytest.mark.gpu
D = 128


def _heads_each(n, n_kv):
    """The launch's rule: heads share their turns while 1024 workgroups are left."""
    sets, each = -(-n // 16), 1
    while each < n_kv and sets * n_kv // (2 * each) >= 1024:
        each *= 2
    return each


# kv heads, tokens of the rows, kv heads of a workgroup: the last one has fewer
# where the heads are no multiple
STEPS = [(32, [900, 0, 300], 2), (32, [1030, 1, 1100, 7], 4), (24, [1500], 2), (9, [3000, 800], 2), (5, [7000], 2), (3, [22000], 4)]


@pytest.mark.parametrize("dtype,layout,part", [
    (torch.float16, "half", 128), (torch.bfloat16, "half", 128), (torch.float16, "half", 50), (torch.bfloat16, "half", 50),
    (torch.float16, "interleaved", 64), (torch.bfloat16, "interleaved", 128), (torch.bfloat16, "half", 16)])
@pytest.mark.parametrize("n_kv,new,each", STEPS)
def test_long_append_is_rotary_and_append(dev, dtype, layout, part, n_kv, new, each):
    print(f"[append4 long] {dtype} {layout} {part} kv {n_kv} {new}", flush=True)
    n = sum(new) + 40                                  # 40 of the rejected row's tokens are in the call
    assert _heads_each(n, n_kv) == each
    g = torch.Generator(device=dev).manual_seed(part + n_kv)
    rot = oi2.Rotary(D, 5e5, rotary_dim=part, layout=layout, device=dev, scaling=SCALINGS[4] if part > 60 else SCALINGS[0])
    rows, n_q = len(new) + 1, n_kv
    pages = sum(-(-(m + 30) // 64) for m in new) + 1
    a, b = (oi2.PagedKVCache(1, n_q, n_kv, rows, max(new) + 100, pages, device=dev, bits=4) for _ in range(2))
    for c in (a, b):
        # pages partly filled before; the last row has too many tokens and is rejected
        first = c.extend([30] * len(new) + [0], c.new_plan(30 * len(new)))
        x = torch.zeros((30 * len(new), n_kv, D), dtype=dtype, device=dev)
        c.append(0, x, x, first)
    step = new + [max(new) + 101]
    pa, pb = (c.extend(step, c.new_plan(sum(step) + 3)) for c in (a, b))
    assert pa.rejected.tolist() == [0] * len(new) + [1]
    qkv = _values(g, (n, n_q + 2 * n_kv, D), dtype, dev)
    q, k, v = qkv[:, :n_q], qkv[:, n_q:n_q + n_kv], qkv[:, n_q + n_kv:]
    qo, q2, k2 = torch.full((n, n_q, D), 3.0, dtype=dtype, device=dev), torch.full((n, n_q, D), 3.0, dtype=dtype, device=dev), torch.zeros_like(k.contiguous())
    a.append(0, k, v, pa, q=q, rotary=rot, q_out=qo)
    rot(q, k, pb.positions[:n], q_out=q2, k_out=k2)
    b.append(0, k2, v, pb)
    assert torch.equal(qo, q2)
    assert torch.equal(a.pages, b.pages)
    assert (a.pages != 0).any(-1).sum() >= sum(-(-m // 64) for m in new) * n_kv
    # odd addresses; k and v of other strides, without q
    a.pages.zero_()
    b.pages.zero_()
    b.append(0, k2, v, pb)
    odd = [torch.empty((n, n_kv, D + 1), dtype=dtype, device=dev)[..., 1:] for _ in range(2)]
    odd[0].copy_(k)
    odd[1].copy_(v)
    a.append(0, *odd, pa, rotary=rot)
    assert torch.equal(a.pages, b.pages)
    a.pages.zero_()
    a.append(0, *(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v)), pa, rotary=rot)
    assert torch.equal(a.pages, b.pages)
