"""The model's path over a 4-bit cache: the layer's counters of parts in a
workspace that the test owns, DecoderStep.forward_paged against its layers one
after the other, a step of chunks and single tokens repeated.
"""
import ctypes

import pytest
import torch

import oi2
from oi2.decode_step import DecoderStep
from oracle import paged as P8
from tests.gpu_helpers import assert_ffn_close
from tests.test_gpu_attention import _cfg, _weights
from tests.test_gpu_decode_step import _layers, dev, split  # noqa: F401

pytestmark = pytest.mark.gpu
H, D, N_Q = 4096, 128, 32


def _items(c, plan, n, max_new):
    """(few, many): numbers of parts of the plan's items, from its work lists."""
    group, rows = c.n_q // c.n_kv, min(c.n_seqs, n)
    cap_append = min(n, n // 64 + 2 * rows, c.n_pages)
    few_only = max_new * group <= 16
    cap_few = rows + (n // (16 // group) if few_only else 0) + (-(-512 // c.n_kv) if c.width > 16 else 0)
    work = plan.work.cpu().numpy()
    few = work[16 + 4 * cap_append:][:16 * work[1]].reshape(-1, 16)
    many = work[16 + 4 * cap_append + 16 * cap_few:][:16 * work[2]].reshape(-1, 16)
    assert all((x[:, 0] < c.n_seqs).all() and (x[:, 7] < x[:, 8]).all() for x in (few, many))
    return few[:, 8], many[:, 8]


@pytest.mark.parametrize("n_kv", [8, 32])
@pytest.mark.parametrize("past,new,few,many", [
    ([3000, 70], [1, 1], True, False),          # parts of few rows
    ([2500, 1300], [3, 130], True, True),       # of 128 rows, beside others
    ([1800, 2600], [90, 1], True, True),
])
def test_layer_clears_its_counters(dev, n_kv, past, new, few, many):
    """The append clears the counters of the attention's parts whatever the
    workspace holds: with all of it 0xFF before every call, and with what the call
    before has left, the output is that of a workspace of zeros."""
    _counters(dev, n_kv, past, new, few, many)


@pytest.mark.parametrize("n_kv,new", [(8, [8, 5]), (8, [7, 1]), (32, [30, 17])])
def test_layer_clears_its_counters_of_two_sets(dev, n_kv, new):
    """Steps of 17 to 32 query rows a row."""
    _counters(dev, n_kv, [2600, 1500], new, min(new) == 1, True)


def _counters(dev, n_kv, past, new, few, many):
    print(f"[kv4 counters] kv {n_kv} {past} + {new}", flush=True)
    g = torch.Generator(device=dev).manual_seed(11)
    attn = oi2.GroupedQueryAttention(0, _weights(dev, n_kv, seed=12), _cfg(n_kv))
    rot = oi2.Rotary(D, 1e4, device=dev)
    c = oi2.PagedKVCache(1, N_Q, n_kv, 2, 3100, sum(P8.pages_of(a + b) for a, b in zip(past, new)), device=dev, bits=4)
    first = c.extend(past, c.new_plan(sum(past)))
    c.append(0, *(torch.randn((sum(past), n_kv, D), generator=g, device=dev).half() for _ in range(2)), first)
    n, lib = sum(new), oi2.load_library()
    plan = c.extend(new, c.new_plan(n, max_new=max(new)))
    parts = _items(c, plan, n, max(new))
    assert [bool((x > 1).any()) for x in parts] == [few, many], parts
    x = torch.randn((n, H), generator=g, device=dev).half()
    ws = torch.zeros(lib.oi2_attn_paged_workspace_bytes(c._ref, plan.max_tokens, plan.max_new, n), dtype=torch.uint8, device=dev)
    outs = []
    for fill in (0, 255, None, 255, 1, None):
        if fill is not None:
            ws.fill_(fill)
        out = torch.full_like(x, 7.0)
        torch.cuda.synchronize()
        assert lib.oi2_kv4_attn_forward(x.data_ptr(), n, ctypes.byref(attn._struct), attn.eps, rot._ref, c._ref, plan._ref, 0, out.data_ptr(),
                                        None, ws.data_ptr(), ws.numel(), torch.cuda.current_stream(dev).cuda_stream or None) == 0
        outs.append(out)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(outs[0]).all()) and bool((outs[0] != 7).any(1).all())
    for i, out in enumerate(outs[1:]):
        assert torch.equal(out, outs[0]), i + 1
    # and the layer's through its module
    assert torch.equal(attn.forward_paged(x, c, plan, rot), outs[0])


@pytest.mark.parametrize("past,new,pad,pages", [
    ([40, 10], [1, 1], 0, 12), ([40, 10, 63], [1, 0, 1], 2, 12), ([150, 64, 9], [1, 1, 1], 1, 5), ([40, 10], [8, 3], 0, 12),
    ([40, 10], [4, 30], 5, 12),
])
def test_step_over_4_bits_equals_its_layers(dev, split, past, new, pad, pages):
    """DecoderStep.forward_paged against the same layers one after the other, each
    with the cold set of the batch of last tokens; a row that the pool has no
    page for among them. Up to 16 tokens the same bits, more at the layers' bar."""
    n = sum(new) + pad
    print(f"[kv4 step] {past} + {new} + {pad}", flush=True)
    g = torch.Generator(device=dev).manual_seed(3)
    prompt = torch.randn((sum(past), H), generator=g, device=dev).half()
    x0 = torch.randn((n, H), generator=g, device=dev).half()
    rot = oi2.Rotary(D, 1e4, device=dev)

    def start():
        attn, ffn = _layers(split, dev)
        c = oi2.PagedKVCache(2, N_Q, 8, len(past), 200, pages, device=dev, bits=4)
        p = c.extend(past, c.new_plan(sum(past)))
        for li in range(2):
            attn[li].forward_paged(prompt, c, p, rot)
        return attn, ffn, c, c.extend(new, c.new_plan(n))

    attn, ffn, c, plan = start()
    y = DecoderStep(attn, ffn).forward_paged(x0, c, plan, rot)
    attn, ffn, c2, plan = start()
    cu, kv = plan.cu.tolist(), plan.kv_len.tolist()
    last = [min(b, n) - 1 for a, b, k in zip(cu, cu[1:], kv) if k > 0 and a < min(b, n)]
    assert (len(last) < sum(t > 0 for t in new)) == (pages == 5)
    x, before = x0, x0
    for li in range(2):
        out = attn[li].forward_paged(x, c2, plan, rot, layer=li)
        x = (x.float() + out.float()).half()
        seen, before = before, x
        x = ffn[li](x[None], ffn[li].submit_cold_fetch(seen[last][:, None]))[0]
    assert torch.equal(c.pages[0], c2.pages[0]) and c.pages[1].any()
    if n <= 16:
        assert torch.equal(y, x) and torch.equal(c.pages, c2.pages)
    else:
        assert_ffn_close(y.float().cpu().numpy(), x.float().cpu().numpy(), what="step over 4 bits")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_chunks_beside_tokens_repeat_themselves(dev, dtype):
    """Ten rows of 1 to 800 tokens over 400 to 9000 positions, tiles of either kind
    cut into parts: call after call the same bits, whatever is in the memory that
    a call's workspace and output get."""
    print(f"[kv4 repeat] {dtype}", flush=True)
    g = torch.Generator(device=dev).manual_seed(5)
    past, new = [400, 9000, 5100, 800, 2500, 6400, 1200, 3300, 450, 7000], [800, 1, 300, 65, 1, 17, 128, 1, 4, 530]
    c = oi2.PagedKVCache(1, N_Q, 8, 10, 9600, sum(P8.pages_of(a + b) for a, b in zip(past, new)), device=dev, bits=4)
    first = c.extend(past, c.new_plan(sum(past)))
    c.append(0, *(torch.randn((sum(past), 8, D), generator=g, device=dev).to(dtype) for _ in range(2)), first)
    plan = c.extend(new, c.new_plan(sum(new), max_new=800))
    c.append(0, *(torch.randn((sum(new), 8, D), generator=g, device=dev).to(dtype) for _ in range(2)), plan)
    assert all((x > 1).any() for x in _items(c, plan, sum(new), 800))
    q = torch.randn((sum(new), N_Q, D), generator=g, device=dev).to(dtype)
    y = c.attend(0, q, plan)
    assert bool(torch.isfinite(y).all())
    for i in range(12):
        junk = torch.full(((1 + i) << 24,), 255 if i % 2 else 1, dtype=torch.uint8, device=dev)
        del junk
        assert torch.equal(c.attend(0, q, plan), y), i


def test_two_captured_steps_over_layers(dev):
    """Two layers over rows cut into parts, captured as a step of single tokens and
    as one of drafts and a chunk, replayed in turn with eager work between:
    every replay equals the same calls made eagerly on a cache of its own."""
    print("[kv4 layer graphs]", flush=True)
    g = torch.Generator(device=dev).manual_seed(23)
    attn = [oi2.GroupedQueryAttention(0, _weights(dev, 8, seed=30 + li), _cfg(8)) for li in range(2)]
    rot = oi2.Rotary(D, 1e4, device=dev)
    past, news = [2500, 63, 1400], [[1, 1, 1], [8, 0, 50]]
    caches = [oi2.PagedKVCache(2, N_Q, 8, 3, 3000, 110, device=dev, bits=4) for _ in range(2)]
    kv = [torch.randn((2, sum(past), 8, D), generator=g, device=dev).half() for _ in range(2)]
    for c in caches:
        p = c.extend(past, c.new_plan(sum(past)))
        for li in range(2):
            c.append(li, kv[li][0], kv[li][1], p, rotary=rot)
    plans = [[c.new_plan(sum(n), max_new=max(n)) for n in news] for c in caches]
    lens = [torch.tensor(n, dtype=torch.int32, device=dev) for n in news]
    xs = [torch.zeros((sum(n), H), dtype=torch.float16, device=dev) for n in news]
    back = torch.tensor(past, dtype=torch.int32, device=dev)

    def step(c, plan, new, x):
        c.extend(new, plan)
        for li in range(2):
            r = torch.empty_like(x)
            attn[li].forward_paged(x, c, plan, rot, layer=li, residual_out=r)
            x = r
        return x

    for i in range(2):                                 # eagerly once: nothing is loaded or set up while capturing
        step(caches[1], plans[1][i], lens[i], xs[i])
    caches[1].rewind(back)
    graphs, outs = [], []
    torch.cuda.synchronize()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(caches[0], plans[0][i], lens[i], xs[i]))
        graphs.append(graph)
    for k in range(12):
        for i in (k % 2, 1 - k % 2):
            xs[i].copy_(torch.randn(xs[i].shape, generator=g, device=dev))
            graphs[i].replay()
            got = outs[i].clone()
            want = step(caches[1], plans[1][i], lens[i], xs[i])
            torch.cuda.synchronize()
            assert torch.equal(got, want) and bool(torch.isfinite(got).all()), (k, i)
            outs[i].zero_()
        if k % 4 == 3:
            for c in caches:
                c.rewind(back)
    # rows of the pool that the eager steps filled before are coded alike
    n = [int(x) for x in caches[0].lens]
    assert n == caches[1].lens.tolist()
    for li in range(2):
        for a, b in zip(*(c.fetch(li, n, sum(n))[:2] for c in caches)):
            assert torch.equal(a, b)
