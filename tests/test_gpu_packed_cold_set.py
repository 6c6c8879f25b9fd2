"""The cold set of a step over the paged cache: predicted from the last token of
every row that is taken and has tokens, as the batch of those tokens predicts it
(engine.py:274-283), and from nothing else in the packed order."""
import os
import tempfile

import pytest
import torch

import oi2
from oi2.decode_step import DecoderStep
from oi2.synth import SyntheticLayer
from tests.gpu_helpers import EPS, assert_ffn_close
from tests.test_gpu_decode_step import _layers, dev, split  # noqa: F401

pytestmark = pytest.mark.gpu
H, D, N_Q = 4096, 128, 32


def _ids(cold):
    counts = cold.counts.cpu().tolist()
    ids = cold.ids.cpu()
    return [i for c, n in enumerate(counts) for i in ids[c * cold.chunk:c * cold.chunk + n].tolist()]


def _last(plan, n):
    """The last token within the first n of every taken row that has one."""
    cu, kv = plan.cu.tolist(), plan.kv_len.tolist()
    return [min(b, n) - 1 for a, b, k in zip(cu, cu[1:], kv) if k > 0 and a < min(b, n)]


# rows, pages, tokens of each row, tokens of x: the pool's end rejects rows
STEPS = [
    (2, 8, [1, 1], 2), (3, 8, [0, 1, 0], 4), (3, 8, [1, 1, 1], 8), (3, 8, [3, 0, 40], 43), (3, 8, [3, 5, 40], 30),
    (3, 2, [2, 30, 70], 102), (3, 2, [2, 30, 70], 110), (4, 2, [70, 1, 70, 70], 220), (130, 130, [1, 0] * 65, 70),
    (2048, 2048, [0] * 2000 + [1] * 48, 48),
]


@pytest.mark.parametrize("rows,pages,new,n", STEPS)
def test_cold_set_is_the_batchs(dev, split, rows, pages, new, n):
    print(f"[cold set] {rows} rows, {n} tokens of {sum(new)}", flush=True)
    g = torch.Generator(device=dev).manual_seed(n)
    _, ffn = _layers(split, dev)
    c = oi2.PagedKVCache(1, N_Q, 8, rows, 128, pages, device=dev)
    plan = c.extend(new, c.new_plan(max(n, sum(new))))
    x = torch.randn((n, H), generator=g, device=dev).half()
    last = _last(plan, n)
    for layer in ffn:
        got = layer.submit_cold_fetch(x, plan).result()
        want = layer.submit_cold_fetch(x[last][:, None]).result()
        assert _ids(got) == _ids(want)
        assert torch.equal(got.counts, want.counts)
    # what stands in the other tokens is not read
    other = torch.ones(n, dtype=torch.bool, device=dev)
    other[last] = False
    for value in (30.0, float("nan")):
        x[other] = value
        assert _ids(ffn[0].submit_cold_fetch(x, plan).result()) == _ids(ffn[0].submit_cold_fetch(x[last][:, None]).result())


def test_no_row_in_the_step(dev, split):
    print("[cold set] no row", flush=True)
    _, ffn = _layers(split, dev)
    c = oi2.PagedKVCache(1, N_Q, 8, 2, 64, 1, device=dev)
    plan = c.extend([0, 0], c.new_plan(4))
    x = torch.full((4, H), float("nan"), dtype=torch.float16, device=dev)
    got = ffn[0].submit_cold_fetch(x, plan).result()
    assert torch.equal(got.counts, ffn[0].submit_cold_fetch(torch.zeros_like(x)[:, None]).result().counts)


def test_cold_set_refusals(dev, split):
    _, ffn = _layers(split, dev)
    c = oi2.PagedKVCache(1, N_Q, 8, 2, 64, 1, device=dev)
    plan = c.new_plan(4)
    x = torch.zeros((5, H), dtype=torch.float16, device=dev)
    with pytest.raises(ValueError):
        ffn[0].submit_cold_fetch(x, plan)
    with pytest.raises(ValueError):
        ffn[0].submit_cold_fetch(x[:4].cpu(), plan)


def _start(split, dev, prompt, lens, pages=12, rows=None, rot=None):
    attn, ffn = _layers(split, dev)
    rot = rot or oi2.Rotary(D, 1e4, device=dev)
    rows = rows or len(lens)
    c = oi2.PagedKVCache(2, N_Q, 8, rows, 200, pages, device=dev)
    p = c.extend(lens, c.new_plan(sum(lens)))
    for li in range(2):
        attn[li].forward_paged(prompt, c, p, rot)
    return attn, ffn, c, rot


@pytest.mark.parametrize("past,new,pad,pages", [
    ([40, 10], [1, 1], 0, 12), ([40, 10], [1, 1], 3, 12), ([40, 10, 63], [1, 0, 1], 2, 12), ([40, 64, 9], [1, 1, 1], 0, 3),
    ([40, 9, 64], [1, 1, 1], 1, 3), ([40, 10], [30, 4], 0, 12), ([40, 10], [4, 30], 5, 12),
])
def test_step_predicts_as_the_batch_does(dev, split, past, new, pad, pages):
    """The loop against the same layers one after the other with the sets of the
    batch of last tokens; rows that the pool has no page for among them (a row
    of 64 positions and a pool of 3 pages)."""
    n = sum(new) + pad
    print(f"[cold set] step {past} + {new} + {pad}", flush=True)
    g = torch.Generator(device=dev).manual_seed(3)
    prompt = torch.randn((sum(past), H), generator=g, device=dev).half()
    x0 = torch.randn((n, H), generator=g, device=dev).half()
    attn, ffn, c, rot = _start(split, dev, prompt, past, pages)
    plan = c.extend(new, c.new_plan(n))
    y = DecoderStep(attn, ffn).forward_paged(x0, c, plan, rot)
    attn, ffn, c, rot = _start(split, dev, prompt, past, pages)
    plan = c.extend(new, c.new_plan(n))
    last = _last(plan, n)
    assert (len(last) < sum(t > 0 for t in new)) == (pages == 3)
    x, before = x0, x0
    for li in range(2):
        out = attn[li].forward_paged(x, c, plan, rot, layer=li)
        x = (x.float() + out.float()).half()
        seen, before = before, x
        x = ffn[li](x[None], ffn[li].submit_cold_fetch(seen[last][:, None]))[0]
    if n <= 16:
        assert torch.equal(y, x)
    else:
        assert_ffn_close(y.float().cpu().numpy(), x.float().cpu().numpy(), what="packed step")


@pytest.mark.parametrize("rejected", [False, True])
def test_padding_and_rejected_rows_have_no_say(dev, split, rejected):
    """What tokens without a position hold changes nothing in the live rows, in a
    captured step's fixed size too."""
    print(f"[cold set] padding, rejected {rejected}", flush=True)
    g = torch.Generator(device=dev).manual_seed(5)
    past, new = ([40, 9, 64], [1, 1, 3]) if rejected else ([40, 9, 64], [1, 1, 0])
    prompt = torch.randn((sum(past), H), generator=g, device=dev).half()
    x = torch.randn((5, H), generator=g, device=dev).half()
    ys = []
    for k in range(3):
        x[2:] = torch.randn((3, H), generator=g, device=dev).half() * 10 ** k
        attn, ffn, c, rot = _start(split, dev, prompt, past, 3)
        plan = c.extend(new, c.new_plan(5))
        assert plan.rejected.tolist() == [0, 0, int(rejected)]
        ys.append(DecoderStep(attn, ffn).forward_paged(x, c, plan, rot)[:2].clone())
    assert torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[2])


def test_requests_in_another_order(dev, split):
    """Two requests swap their rows: so do their outputs."""
    print("[cold set] order", flush=True)
    g = torch.Generator(device=dev).manual_seed(7)
    a, b = (torch.randn((m, H), generator=g, device=dev).half() for m in (40, 10))
    x = torch.randn((2, H), generator=g, device=dev).half()
    ys = []
    for prompt, lens, xs in ((torch.cat([a, b]), [40, 10], x), (torch.cat([b, a]), [10, 40], x.flip(0))):
        attn, ffn, c, rot = _start(split, dev, prompt, lens)
        ys.append(DecoderStep(attn, ffn).forward_paged(xs, c, c.extend([1, 1], c.new_plan(2)), rot))
    assert_ffn_close(ys[1].flip(0).float().cpu().numpy(), ys[0].float().cpu().numpy(), tol=1e-3, cos_min=0.999999, what="order")


def test_a_captured_step_whose_requests_end(dev, split):
    """A step of three rows captured once; rows leave it between the replays, and
    the tokens behind the last one hold what they held: every replay equals an
    eager step."""
    print("[cold set] graph", flush=True)
    g = torch.Generator(device=dev).manual_seed(9)
    past = [62, 30, 38]
    prompt = torch.randn((sum(past), H), generator=g, device=dev).half()
    tokens = [torch.randn((3, H), generator=g, device=dev).half() for _ in range(4)]
    news = [torch.tensor(v, dtype=torch.int32, device=dev) for v in ([1, 1, 1], [1, 0, 1], [0, 0, 1], [0, 1, 0])]
    stream = torch.cuda.Stream(device=dev)
    with torch.cuda.stream(stream):
        attn, ffn, c, rot = _start(split, dev, prompt, past)
        step, plan, eager = DecoderStep(attn, ffn), c.new_plan(3, max_new=1), []
        for x, new in zip(tokens, news):
            c.extend(new, plan)
            eager.append(step.forward_paged(x, c, plan, rot).clone())
        attn, ffn, cg, rot = _start(split, dev, prompt, past)
        step, pg = DecoderStep(attn, ffn), cg.new_plan(3, max_new=1)
        x_in, new_in = tokens[0].clone(), news[0].clone()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        cg.extend(new_in, pg)
        y = step.forward_paged(x_in, cg, pg, rot)
    other = torch.randn((512, 512), generator=g, device=dev)
    for i, (x, new) in enumerate(zip(tokens, news)):
        x_in.copy_(x)
        new_in.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager[i]), f"replay {i}"
        other = (other @ other).tanh()
        torch.cuda.synchronize()
    assert torch.equal(cg.pages, c.pages)
    del graph


def test_cold_set_from_files(dev):
    """Records read from the split file: the same set from the same rows."""
    print("[cold set] file", flush=True)
    g = torch.Generator(device=dev).manual_seed(11)
    inter = 2048
    lay = SyntheticLayer(g, inter, 500, device=dev, with_predictor=True, pred_dtype=torch.float32)
    with tempfile.TemporaryDirectory(dir=os.path.dirname(os.path.abspath(__file__))) as tmp:
        for d in ("hot", "pred"):
            os.makedirs(os.path.join(tmp, d))
        lay.hot.save(os.path.join(tmp, "hot", "layer_000_expert_000.pt"))
        lay.predictor.save(os.path.join(tmp, "pred", "layer_000_expert_000.pt"))
        paths = [os.path.join(tmp, f) for f in ("cold_weights.bin", "cold_index.npy")]
        w = oi2.format.ColdFileWriter(paths[0], 1)
        w.add_section(0, lay.records.cpu().numpy())
        w.close(paths[1])
        cfg = {"hidden_dim": H, "intermediate_dim": inter, "hidden_act": "silu", "act_on_both": False, "rms_norm_eps": EPS,
               "num_experts": 1}
        reg = oi2.PredictorRegistry(os.path.join(tmp, "pred"), device=dev)
        stores = [oi2.ColdWeightStore(*paths, cfg, device=dev, **kw) for kw in ({"residency": "file"}, {})]
        try:
            lf, lh = (oi2.SparseFFNLayer(0, os.path.join(tmp, "hot"), s, reg, cfg, dev, None, ffn_norm_weight=lay.norm_w.cpu())
                      for s in stores)
            c = oi2.PagedKVCache(1, N_Q, 8, 3, 64, 2, device=dev)
            plan = c.extend([2, 1, 1], c.new_plan(6))
            assert plan.rejected.tolist() == [0, 0, 1]
            x = torch.randn((6, H), generator=g, device=dev).half()
            staged, held = lf.submit_cold_fetch(x, plan).result(), lh.submit_cold_fetch(x, plan).result()
            want = lf.submit_cold_fetch(x[[1, 2]][:, None]).result()
            torch.cuda.synchronize()
            assert staged.count() == held.count() == want.count() > 0
            assert torch.equal(staged.section.records, want.section.records)
            y, z = lf(x[None], lf.submit_cold_fetch(x, plan)), lh(x[None], lh.submit_cold_fetch(x, plan))
            torch.cuda.synchronize()
            assert_ffn_close(y.float().cpu().numpy(), z.float().cpu().numpy(), tol=2e-3, cos_min=0.99999, what="file")
        finally:
            for s in stores:
                s.close()


@pytest.mark.parametrize("pad", [1, 12, 37, 100])
def test_padding_that_is_not_finite_harms_no_row(dev, split, pad):
    """Tokens without a position hold NaN and infinities: the live rows' results
    keep their bits (up to 16 tokens, whose FFN sums are in a fixed order) or the
    FFN's bar."""
    print(f"[cold set] padding of {pad} that is not finite", flush=True)
    g = torch.Generator(device=dev).manual_seed(13)
    past, new = [40, 9], [2, 1]
    prompt = torch.randn((sum(past), H), generator=g, device=dev).half()
    x = torch.randn((3 + pad, H), generator=g, device=dev).half()
    ys = []
    for bad in (0.0, float("nan"), float("inf")):
        if bad:
            x[3:] = bad
        attn, ffn, c, rot = _start(split, dev, prompt, past)
        plan = c.extend(new, c.new_plan(3 + pad))
        ys.append(DecoderStep(attn, ffn).forward_paged(x, c, plan, rot)[:3].clone())
    for y in ys[1:]:
        if pad <= 13:
            assert torch.equal(y, ys[0])
        else:
            assert_ffn_close(y.float().cpu().numpy(), ys[0].float().cpu().numpy(), tol=1e-3, cos_min=0.999999, what="padding")
