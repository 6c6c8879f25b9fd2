"""The model's path over the paged cache: GroupedQueryAttention.forward_paged
and DecoderStep.forward_paged, the step captured into a graph, and the cache on
other streams.

A layer's k and v codes are compared bit for bit with append's of the same
projections; its output with the float64 chain of the reference's attention
(engine.py:90-125) at the reference layer's bar (max rel err 1e-2, cosine >=
0.9999) over the positions that the cache holds, so that the codes' rounding is
on both sides.
"""
import numpy as np
import pytest
import torch

import oi2
from oi2.decode_step import DecoderStep
from oracle import oracle as O
from oracle import paged as P
from tests.gpu_helpers import EPS, assert_ffn_close
from tests.test_gpu_attention import _cfg, _dense, _weights
from tests.test_gpu_decode_step import _layers, _stack, dev, split  # noqa: F401

pytestmark = pytest.mark.gpu
H, D, N_Q = 4096, 128, 32


def _x(g, n, dev):
    return torch.randn((n, H), generator=g, device=dev).half()


def _plain_kv(w, n_kv, x):
    """k and v (tokens, n_kv, 128) of x's rows, not rotated: the layer's own
    cache under tables of cosine 1 and sine 0."""
    n = x.shape[0]
    one, zero = torch.ones((n, D // 2), device=x.device), torch.zeros((n, D // 2), device=x.device)
    _, (k, v) = oi2.GroupedQueryAttention(0, w, _cfg(n_kv))(x[None], one, zero)
    return k[0].transpose(0, 1), v[0].transpose(0, 1)


@pytest.mark.parametrize("n_kv", [8, 32])
@pytest.mark.parametrize("past,new", [([5], [1]), ([200, 64, 7], [1, 1, 1]), ([0, 130, 63, 9, 1], [1, 2, 0, 1, 1]),
                                      ([0, 300], [70, 1]), ([40, 0, 100], [3, 190, 1])])
def test_layer_over_pages(dev, n_kv, past, new):
    print(f"[paged layer] kv {n_kv} {past} + {new}", flush=True)
    g = torch.Generator(device=dev).manual_seed(11)
    w = _weights(dev, n_kv, seed=12)
    rows, n_pages = len(past), sum(P.pages_of(a + b) for a, b in zip(past, new))
    attn = oi2.GroupedQueryAttention(0, w, _cfg(n_kv))
    rot = oi2.Rotary(D, 1e4, device=dev)
    caches = [oi2.PagedKVCache(2, N_Q, n_kv, rows, 400, n_pages, device=dev) for _ in range(2)]
    o = P.Cache(rows, 400, n_pages, n_kv)
    wq, _, _, wo, nw = _dense(w)
    for step in (past, new):
        n = sum(step)
        plans = [c.new_plan(n + 3, max_new=max(step)) for c in caches]
        for c, p in zip(caches, plans):
            c.extend(step, p)
        ref = o.extend(step, n + 3, max(step))
        x = _x(g, n + 3, dev)
        resid = torch.empty_like(x)
        out = attn.forward_paged(x, caches[0], plans[0], rot, layer=1, residual_out=resid)
        assert torch.equal(resid, (x.float() + out.float()).half())
        assert not out[n:].any()                    # tokens without a position
        # n + 3 rows take the same projection kernels
        k, v = _plain_kv(w, n_kv, x)
        caches[1].append(1, k, v, plans[1], rotary=rot)
        for a, b in zip(caches[0].codes(1) + caches[0].scales(1), caches[1].codes(1) + caches[1].scales(1)):
            assert torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a,
                               b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)
        assert not caches[0].pages[0].any()
        # the chain, over what the cache holds
        for i, (codes, scale) in enumerate(zip(caches[0].codes(1), caches[0].scales(1))):
            o.codes[i] = codes.contiguous().view(n_pages, n_kv, 64, D).float().cpu().numpy().astype(np.float64)
            o.exps[i] = np.log2(scale.abs().double().cpu().numpy()).astype(np.int64)
        if not n:
            continue
        xn = O.f16(O.rmsnorm(x[:n].float().cpu().numpy().astype(np.float64), nw, EPS))
        q = O.f16(xn @ wq.T).reshape(n, N_Q, D)
        q = O.f16(P.rotate(q, ref["positions"][:n], oi2.rotary_frequencies(D, 1e4)[0], 1.0, "half"))
        a = O.f16(o.attend(q, ref, D ** -0.5)[0]).reshape(n, H)
        assert_ffn_close(out[:n].float().cpu().numpy(), O.f16(a @ wo.T), what="paged layer")


def test_layer_rejected_rows_and_no_tokens(dev):
    """A row that the pool has no page for: its tokens give 0 and leave the
    cache; the others' are what they are without it."""
    g = torch.Generator(device=dev).manual_seed(21)
    w = _weights(dev, 8, seed=22)
    attn = oi2.GroupedQueryAttention(0, w, _cfg(8))
    rot = oi2.Rotary(D, 1e4, device=dev)
    x = _x(g, 40, dev)
    for n in (4, 40):
        print(f"[paged layer] rejected row, {n} tokens", flush=True)
        new = [2, 1, n - 3]
        c, full = (oi2.PagedKVCache(1, N_Q, 8, 3, 64, pages, device=dev) for pages in (2, 3))
        p, pf = c.new_plan(40), full.new_plan(40)
        c.extend(new, p)
        full.extend(new, pf)
        assert p.rejected.tolist() == [0, 0, 1] and pf.rejected.tolist() == [0, 0, 0]
        y, yf = attn.forward_paged(x[:n], c, p, rot), attn.forward_paged(x[:n], full, pf, rot)
        assert torch.equal(y[:3], yf[:3]) and not y[3:].any() and yf[3:].any()
    assert attn.forward_paged(x[:0], c, p, rot).shape == (0, H)


def test_layer_refusals(dev):
    w = _weights(dev, 8, seed=31)
    attn = oi2.GroupedQueryAttention(0, w, _cfg(8))
    rot = oi2.Rotary(D, 1e4, device=dev)
    c = oi2.PagedKVCache(1, N_Q, 8, 2, 64, 2, device=dev)
    other = oi2.PagedKVCache(1, N_Q, 4, 2, 64, 2, device=dev)
    p = c.new_plan(4)
    x = torch.zeros((4, H), dtype=torch.float16, device=dev)
    bad = [(TypeError, (x.bfloat16(), c, p, rot), {}), (TypeError, (x[None], c, p, rot), {}),
           (ValueError, (x, other, other.new_plan(4), rot), {}), (ValueError, (x, c, other.new_plan(4), rot), {}),
           (ValueError, (x, c, p, oi2.Rotary(64, 1e4, device=dev)), {}), (ValueError, (x, c, p, rot), {"layer": 1}),
           (ValueError, (torch.cat([x, x]), c, p, rot), {}), (ValueError, (x.cpu(), c, p, rot), {}),
           (ValueError, (x, c, p, rot), {"residual_out": x[:2]}),
           (ValueError, (x, c, p, rot), {"residual_out": x.float()})]
    for i, (err, args, kw) in enumerate(bad):
        print(f"[paged layer] refusal {i}", flush=True)
        with pytest.raises(err):
            attn.forward_paged(*args, **kw)
    with pytest.raises(ValueError):
        DecoderStep([attn], [None]).forward_paged(x[None], c, p, rot)
    with pytest.raises(ValueError):
        DecoderStep([attn, attn], [None, None]).forward_paged(x, c, p, rot)


@pytest.mark.parametrize("new", [[1, 0], [1, 1], [30, 4]])
def test_step_equals_plain_loop(dev, split, new):
    """The step's loop against the same layers one after the other, each
    prediction made from the same state just before its FFN: the same bits (16
    tokens' FFN sums are in a fixed order, more are compared at its bar)."""
    n = sum(new)
    print(f"[paged step] {new}", flush=True)
    g = torch.Generator(device=dev).manual_seed(41)
    x0, prompt = _x(g, n, dev), _x(g, 90, dev)
    rot = oi2.Rotary(D, 1e4, device=dev)
    results = []
    for plain in (False, True):
        attn, ffn = _layers(split, dev)
        c = oi2.PagedKVCache(2, N_Q, 8, 2, 200, 6, device=dev)
        p = c.extend([80, 10], c.new_plan(90))
        for li in range(2):
            attn[li].forward_paged(prompt, c, p, rot)
        p = c.extend(new, c.new_plan(n))
        if not plain:
            results.append((DecoderStep(attn, ffn).forward_paged(x0, c, p, rot), c))
            continue
        x, before = x0, x0
        for li in range(2):
            out = attn[li].forward_paged(x, c, p, rot, layer=li)
            x = (x.float() + out.float()).half()
            seen, before = before, x
            x = ffn[li](x[None], ffn[li].submit_cold_fetch(seen[None]))[0]
        results.append((x, c))
    (y, c), (yr, cr) = results
    if n <= 16:
        assert torch.equal(y, yr)
        assert torch.equal(c.pages, cr.pages)
    else:
        assert_ffn_close(y.float().cpu().numpy(), yr.float().cpu().numpy(), what="paged step")


def test_stack_step_equals_layers(dev, split):
    print("[paged step] stack", flush=True)
    g = torch.Generator(device=dev).manual_seed(51)
    x0 = _x(g, 1, dev)
    rot = oi2.Rotary(D, 1e4, device=dev)
    ys = []
    for stacked in (False, True):
        attn, ffn = _layers(split, dev)
        c = oi2.PagedKVCache(2, N_Q, 8, 1, 100, 2, device=dev)
        step = DecoderStep(attn, _stack(split) if stacked else ffn)
        plan, x = c.new_plan(1), x0
        for _ in range(3):
            c.extend([1], plan)
            x = step.forward_paged(x, c, plan, rot)
        ys.append(x.clone())
        if stacked:
            with pytest.raises(ValueError):
                step.forward_paged(x0.repeat(2, 1), c, c.new_plan(2), rot)
            torch.cuda.synchronize()
            step.ffn_layers.close()
    assert torch.equal(*ys)


def test_captured_steps_equal_eager_steps(dev, split):
    """A decoding step of three rows (extend and both layers) captured once and
    replayed: each replay takes the next token of every row, as an eager run
    over a cache of its own does, with eager work between."""
    print("[paged step] graph", flush=True)
    g = torch.Generator(device=dev).manual_seed(61)
    rot = oi2.Rotary(D, 1e4, device=dev)
    prompt, tokens = _x(g, 400, dev), [_x(g, 3, dev) for _ in range(5)]
    new = torch.ones(3, dtype=torch.int32, device=dev)
    attn, ffn = _layers(split, dev)
    step = DecoderStep(attn, ffn)
    stream = torch.cuda.Stream(device=dev)

    def start():
        c = oi2.PagedKVCache(2, N_Q, 8, 3, 500, 10, device=dev)
        p = c.extend([62, 300, 38], c.new_plan(400))
        for li in range(2):
            attn[li].forward_paged(prompt, c, p, rot, layer=li)
        return c, c.new_plan(3, max_new=1)

    with torch.cuda.stream(stream):
        c, plan = start()
        eager = []
        for x in tokens:
            c.extend(new, plan)
            eager.append(step.forward_paged(x, c, plan, rot).clone())
        cg, pg = start()
        x_in = tokens[0].clone()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        cg.extend(new, pg)
        y = step.forward_paged(x_in, cg, pg, rot)
    other = torch.randn((512, 512), generator=g, device=dev)
    for i, x in enumerate(tokens):
        x_in.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager[i]), f"replay {i} differs from the eager step"
        other = (other @ other).tanh()
        torch.cuda.synchronize()
    assert torch.equal(cg.pages, c.pages) and torch.equal(cg.lens, c.lens)
    del graph


@pytest.mark.parametrize("past,new", [([900, 3, 64], [1, 1, 1]), ([3000, 10, 200], [1, 300, 4])])
def test_captured_operators(dev, past, new):
    """Table, append, attention and the cut back in one graph, many parts a row
    among them: every replay the eager bits."""
    print(f"[paged graph] {past} + {new}", flush=True)
    g = torch.Generator(device=dev).manual_seed(71)
    rot = oi2.Rotary(D, 1e4, device=dev)
    n = sum(new)

    def data(m, heads):
        return torch.randn((m, heads, D), generator=g, device=dev).half()

    first, ins = (data(sum(past), 8), data(sum(past), 8)), [(data(n, 8), data(n, 8), data(n, N_Q)) for _ in range(4)]
    lens, back = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (new, past))
    stream = torch.cuda.Stream(device=dev)

    def start():
        c = oi2.PagedKVCache(1, N_Q, 8, 3, 4000, 80, device=dev)
        c.append(0, *first, c.extend(past, c.new_plan(sum(past))))
        return c, c.new_plan(n, max_new=max(new))

    def run(c, p, k, v, q):
        c.extend(lens, p)
        y = c.attend(0, c.append(0, k, v, p, q=q, rotary=rot), p)
        c.rewind(back)
        return y

    with torch.cuda.stream(stream):
        c, p = start()
        want = [run(c, p, *x) for x in ins]
        assert not torch.equal(want[0], want[1])
        cg, pg = start()
        static = [x.clone() for x in ins[0]]
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = run(cg, pg, *static)
    other = torch.randn((512, 512), generator=g, device=dev)
    for i, x in enumerate(ins):
        for a, b in zip(static, x):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i]), f"replay {i}"
        other = (other @ other).tanh()
        torch.cuda.synchronize()
    assert torch.equal(cg.pages, c.pages) and torch.equal(cg.n_free, c.n_free)
    del graph


def test_two_caches_on_two_streams(dev):
    """Steps of two caches on streams of their own, under way together, against
    the same on the default stream."""
    print("[paged streams]", flush=True)
    g = torch.Generator(device=dev).manual_seed(81)
    rot = oi2.Rotary(D, 1e4, device=dev)
    past, new = [5000, 700], [1, 40]
    data = [[torch.randn((m, h, D), generator=g, device=dev).bfloat16() for m, h in
             ((sum(past), 8), (sum(past), 8), (41, 8), (41, 8), (41, N_Q))] for _ in range(2)]

    def run(k0, v0, k, v, q):
        c = oi2.PagedKVCache(1, N_Q, 8, 2, 6000, 100, device=dev)
        c.append(0, k0, v0, c.extend(past, c.new_plan(sum(past))))
        p = c.extend(new, c.new_plan(41))
        q = c.append(0, k, v, p, q=q, rotary=rot)
        return [c.attend(0, q, p) for _ in range(4)]

    want = [run(*d)[0] for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    got = []
    for s, d in zip(streams, data):
        with torch.cuda.stream(s):
            got.append(run(*d))
    torch.cuda.synchronize()
    for y, ys in zip(want, got):
        assert all(torch.equal(y, x) for x in ys)
