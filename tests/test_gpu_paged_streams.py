"""Attention calls of one step's plan that run at the same time: other layers,
other queries, on two streams and in two graphs; workspaces that hold anything."""
import ctypes

import pytest
import torch

import oi2
from oi2 import _lib
from tests.test_gpu_paged import dev  # noqa: F401

pytestmark = pytest.mark.gpu
D, N_Q, N_KV = 128, 32, 8
# rows whose pages are cut into parts: few query rows, many, and both
STEPS = [([9000, 300, 5000], [1, 1, 1]), ([6000], [300]), ([7000, 20, 4000], [2, 250, 1])]


def _cache(dev, past, new, seed=1):
    g = torch.Generator(device=dev).manual_seed(seed)

    def data(n, heads):
        return torch.randn((n, heads, D), generator=g, device=dev).half()

    c = oi2.PagedKVCache(2, N_Q, N_KV, len(past), 10000, 400, device=dev)
    first = c.extend(past, c.new_plan(sum(past)))
    for li in range(2):
        c.append(li, data(sum(past), N_KV), data(sum(past), N_KV), first)
    plan = c.extend(new, c.new_plan(sum(new), max_new=max(new)))
    for li in range(2):
        c.append(li, data(sum(new), N_KV), data(sum(new), N_KV), plan)
    return c, plan, [data(sum(new), N_Q) for _ in range(2)]


@pytest.mark.parametrize("past,new", STEPS)
def test_layers_of_a_step_on_two_streams(dev, past, new):
    print(f"[paged streams] {past} + {new}", flush=True)
    c, plan, q = _cache(dev, past, new)
    want = [c.attend(li, q[li], plan) for li in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    got = [[], []]
    for _ in range(30):
        for li, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[li].append(c.attend(li, q[li], plan))
    torch.cuda.synchronize()
    for li in range(2):
        assert all(torch.equal(y, want[li]) for y in got[li])


def test_graphs_of_a_step_replayed_together(dev):
    print("[paged streams] two graphs", flush=True)
    past, new = STEPS[0]
    c, plan, q = _cache(dev, past, new)
    want = [c.attend(li, q[li], plan) for li in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    graphs, outs = [], []
    for li, s in enumerate(streams):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            outs.append(c.attend(li, q[li], plan))
    other = torch.randn((512, 512), device=dev)
    for _ in range(10):
        for li, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[li].replay()
        eager = c.attend(0, q[0], plan)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])
        other = (other @ other).tanh()
        for y in outs:
            y.zero_()
        torch.cuda.synchronize()
    graphs.clear()


@pytest.mark.parametrize("past,new", STEPS)
def test_workspaces_may_hold_anything(dev, past, new):
    """Through the C ABI: a workspace of zeros, of ones and of what another call
    left; the plan's memory stays as extend left it."""
    print(f"[paged workspace] {past} + {new}", flush=True)
    c, plan, q = _cache(dev, past, new)
    lib = oi2.load_library()
    want = c.attend(0, q[0], plan)
    nbytes = lib.oi2_kv_attend_workspace_bytes(c._ref, plan.max_tokens, plan.max_new)
    ws = torch.zeros(nbytes, dtype=torch.uint8, device=dev)
    work = plan.work.clone()
    x, h = _lib.heads(q[0], N_Q)
    for fill in (0, 255, 1, None):
        if fill is not None:
            ws.fill_(fill)
        out = torch.empty_like(want)
        _lib.check(lib.oi2_kv_attend(c._ref, plan._ref, 0, _lib.DTYPE_F16, x.shape[0], ctypes.byref(h), D ** -0.5, out.data_ptr(),
                                     ws.data_ptr(), nbytes, _lib.stream_handle(dev)))
        assert torch.equal(out, want)
    assert torch.equal(plan.work, work)
