"""Outputs that are the inputs themselves, and outputs beside them in one buffer."""
import pytest
import torch

import oi2
from tests.test_gpu_attention import _cfg, _weights
from tests.test_gpu_paged import dev  # noqa: F401

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("past,new", [([700, 3], [1, 1]), ([9000], [3]), ([3000, 60], [300, 20])])
def test_attend_into_its_query(dev, dtype, past, new):
    print(f"[in place] {dtype} {past} + {new}", flush=True)
    g = torch.Generator(device=dev).manual_seed(1)
    c = oi2.PagedKVCache(1, 8, 2, len(past), 10000, 200, device=dev)
    for lens in (past, new):
        plan = c.extend(lens, c.new_plan(sum(lens)))
        k, v = (torch.randn((sum(lens), 2, D), generator=g, device=dev).to(dtype) for _ in range(2))
        c.append(0, k, v, plan)
    n = sum(new)
    q = torch.randn((n, 8, D), generator=g, device=dev).to(dtype)
    want = c.attend(0, q, plan)
    for _ in range(5):
        x = q.clone()
        assert c.attend(0, x, plan, out=x) is x and torch.equal(x, want)
    both = torch.cat([q, q])
    c.attend(0, both[:n], plan, out=both[n:])
    assert torch.equal(both[:n], q) and torch.equal(both[n:], want)
    if n > 1:
        with pytest.raises(Exception, match="shares memory"):
            c.attend(0, both[:n], plan, out=both[1:n + 1])


def test_rotary_and_append(dev):
    rot = oi2.Rotary(D, 1e4, device=dev)
    c = oi2.PagedKVCache(1, 8, 8, 1, 100, 2, device=dev)
    plan = c.extend([30], c.new_plan(30))
    q, k = (torch.randn(30, 8, D, device=dev).half() for _ in range(2))
    want = rot(q, k, plan.positions)
    x, y = q.clone(), k.clone()
    rot(x, y, plan.positions, q_out=x, k_out=y)
    assert torch.equal(x, want[0]) and torch.equal(y, want[1])
    for kw in (dict(q_out=k), dict(k_out=q), dict(q_out=y, k_out=y)):
        with pytest.raises(Exception, match="shares memory"):
            rot(q, k, plan.positions, **kw)
    for out in (k, q.view(-1)[:30 * 8 * D].view(30, 8, D)):
        if out is k:
            with pytest.raises(Exception, match="shares memory"):
                c.append(0, k, k, plan, q=q, rotary=rot, q_out=out)
        else:
            assert torch.equal(c.append(0, k, k, plan, q=q, rotary=rot, q_out=out), want[0])


@pytest.mark.parametrize("n", [1, 5, 40])
def test_layer_residual_into_its_input(dev, n):
    print(f"[in place] layer {n}", flush=True)
    attn = oi2.GroupedQueryAttention(0, _weights(dev, 8, seed=2), _cfg(8))
    rot = oi2.Rotary(D, 1e4, device=dev)
    g = torch.Generator(device=dev).manual_seed(2)
    buf = torch.randn((n + 1, 4096), generator=g, device=dev).half()
    got = []
    for into in (False, True):
        c = oi2.PagedKVCache(1, 32, 8, 1, 64, 1, device=dev)
        plan = c.extend([n], c.new_plan(n))
        x = buf[:n].clone()
        resid = x if into else torch.empty_like(x)
        attn.forward_paged(x, c, plan, rot, residual_out=resid)
        got.append(resid)
    assert torch.equal(*got)
    if n > 1:
        with pytest.raises(ValueError):
            attn.forward_paged(buf[:n], c, plan, rot, residual_out=buf[1:])


def test_one_head_in_place(dev):
    """A tensor of one head is dense whatever its stride of heads says."""
    rot = oi2.Rotary(D, 1e4, device=dev)
    x = torch.randn(9, D, device=dev).half()
    pos = torch.arange(9, device=dev, dtype=torch.int32)
    want = rot(x[:, None], None, pos)[0]
    q = x.clone().as_strided((9, 1, D), (D, 999, 1))
    assert q.is_contiguous() and rot(q, None, pos, q_out=q)[0] is q and torch.equal(q, want)
    c = oi2.PagedKVCache(1, 1, 1, 1, 64, 1, device=dev)
    plan = c.extend([9], c.new_plan(9))
    k = torch.randn(9, 1, D, device=dev).half()
    c.append(0, k, k, plan)
    y = c.attend(0, q, plan)
    assert c.attend(0, q, plan, out=q) is q and torch.equal(q, y)
