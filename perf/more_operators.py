"""Serving on a paged 4-bit KV cache: what is measured of it.

Three operators, each as a serving loop calls it, on the attention geometry that
the framework serves (query heads of 128, groups of 1 to 8 of them per kv head):

  store    k and v of a step coded into their pages, q and k rotated on the way
           where the model's projections leave that to the cache, and what the
           cache then stands for read back, as a prompt's own dense attention
           takes it
  read     positions of many rows read back as dense k and v: a request that
           is moved away, a prefix that another engine takes over
  attend   attention of a step's query tokens over the cache

The cache's pages hold 64 positions.  A head's 128 values are four groups of
32; a group is 32 whole numbers in [-7, 7] times a scale, its largest magnitude
over 7 rounded to 8 significant bits (a multiple of 2^-24, at most 9344).

With ``own`` false they are computed by elementary torch operations in 32 bits
(rotations in 64); with ``own`` true by ``oi2.PagedKVCache(bits=4)``.
"""
import math
import os
import sys

import torch

own = False

N_Q = 32
HEAD = 128
GROUP = 32
PAGE = 64
TOP_CODE = 7
TOP_SCALE = 9344.0
LEAST_SCALE = 2.0 ** -24
THETA = 500000.0
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ── the cases ────────────────────────────────────────────────────────────────

def listed():
    return [
        # a decoding step of 24 chats: one token each into pages partly filled
        {"name": "store_step_24", "op": "store", "seqs": 24, "past_lo": 30, "past_hi": 900, "new_lo": 1, "new_hi": 1,
         "idle": 0, "n_kv": 8, "dtype": "fp16", "rotate": "half", "part": 128},
        # prompts of several requests, odd lengths, whose projections rotate q and k themselves
        {"name": "store_prompts_6", "op": "store", "seqs": 6, "past_lo": 1, "past_hi": 300, "new_lo": 400, "new_hi": 2600,
         "idle": 0, "n_kv": 8, "dtype": "bf16", "rotate": "none", "part": 0},
        # drafts of five tokens of a model with a kv head for each query head, half of the head rotated in pairs
        {"name": "store_drafts_33", "op": "store", "seqs": 33, "past_lo": 5, "past_hi": 400, "new_lo": 5, "new_hi": 5,
         "idle": 0, "n_kv": 32, "dtype": "fp16", "rotate": "interleaved", "part": 64},
        # one preempted chat leaves the GPU
        {"name": "read_chat_1", "op": "read", "seqs": 1, "past_lo": 900, "past_hi": 900, "count_lo": 900, "count_hi": 900,
         "n_kv": 8, "dtype": "fp16"},
        # a server is drained: every position of requests of many lengths
        {"name": "read_all_48", "op": "read", "seqs": 48, "past_lo": 100, "past_hi": 6000, "count_lo": 6000, "count_hi": 6000,
         "n_kv": 8, "dtype": "bf16"},
        # the last positions of long contexts, few kv heads
        {"name": "read_ends_12", "op": "read", "seqs": 12, "past_lo": 700, "past_hi": 30000, "count_lo": 50, "count_hi": 900,
         "n_kv": 4, "dtype": "fp16"},
        # the smallest: one chat's next token
        {"name": "attend_step_1", "op": "attend", "seqs": 1, "past_lo": 1100, "past_hi": 1100, "new_lo": 1, "new_hi": 1,
         "idle": 0, "n_kv": 8, "dtype": "fp16"},
        # a server's decoding step: ragged long contexts, a padded batch with idle rows
        {"name": "attend_step_48", "op": "attend", "seqs": 48, "past_lo": 500, "past_hi": 20000, "new_lo": 1, "new_hi": 1,
         "idle": 6, "n_kv": 8, "dtype": "fp16"},
        # two sequences over very long contexts, eight query heads a kv head
        {"name": "attend_long_2", "op": "attend", "seqs": 2, "past_lo": 60000, "past_hi": 150000, "new_lo": 1, "new_hi": 1,
         "idle": 0, "n_kv": 4, "dtype": "bf16"},
        # drafts of four tokens checked together
        {"name": "attend_drafts_20", "op": "attend", "seqs": 20, "past_lo": 200, "past_hi": 7000, "new_lo": 4, "new_hi": 4,
         "idle": 0, "n_kv": 8, "dtype": "bf16"},
        # a whole prompt at once, no cache before it
        {"name": "attend_prompt_4100", "op": "attend", "seqs": 1, "past_lo": 0, "past_hi": 0, "new_lo": 4100, "new_hi": 4100,
         "idle": 0, "n_kv": 8, "dtype": "fp16"},
        # chunks of prompts on their caches beside single decoding tokens
        {"name": "attend_mixed_10", "op": "attend", "seqs": 10, "past_lo": 400, "past_hi": 9000, "new_lo": 1, "new_hi": 800,
         "idle": 0, "n_kv": 8, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _range(rng, lo, hi):
    a, b = sorted((_log_int(rng, lo, hi), _log_int(rng, lo, hi)))
    return a, b


def draw(rng):
    op = rng.choice(["store", "store", "read", "attend", "attend", "attend"])
    dtype, n_kv = rng.choice(["fp16", "bf16"]), rng.choice([4, 8, 8, 16, 32])
    if op == "store":
        a, b = _range(rng, 1, 600)
        lo, hi = rng.choice([(1, 1), (2, 6), _range(rng, 10, 2000)])
        seqs = _log_int(rng, 1, max(1, min(64, 9000 // hi)))
        rotate = rng.choice(["none", "half", "half", "interleaved"])
        return {"op": op, "seqs": seqs, "past_lo": a, "past_hi": b, "new_lo": lo, "new_hi": hi, "idle": rng.choice([0, 4]),
                "n_kv": n_kv, "dtype": dtype, "rotate": rotate, "part": 0 if rotate == "none" else rng.choice([32, 64, 96, 128, 128])}
    if op == "read":
        a, b = _range(rng, 10, 20000)
        lo, hi = rng.choice([(b, b), _range(rng, 1, b)])
        seqs = _log_int(rng, 1, max(1, min(64, 1000000 // (b * n_kv))))
        return {"op": op, "seqs": seqs, "past_lo": a, "past_hi": b, "count_lo": lo, "count_hi": hi, "n_kv": n_kv, "dtype": dtype}
    kind = rng.choice(["step", "step", "drafts", "prompt", "mixed"])
    if kind in ("step", "drafts"):
        a, b = _range(rng, 50, 40000)
        lo, hi = (1, 1) if kind == "step" else (2, rng.choice([3, 5, 8]))
        seqs = _log_int(rng, 1, max(1, min(56, 1800000 // (b * n_kv))))
    elif kind == "prompt":
        a, b = 0, 0
        lo, hi = _range(rng, 20, 3000)
        seqs = _log_int(rng, 1, max(1, min(8, (3000 // hi) ** 2)))
    else:
        a, b = _range(rng, 100, 8000)
        lo, hi = 1, _log_int(rng, 30, 700)
        seqs = rng.randint(2, 8)
    return {"op": op, "seqs": seqs, "past_lo": a, "past_hi": b, "new_lo": lo, "new_hi": hi, "idle": rng.choice([0, 3]),
            "n_kv": n_kv, "dtype": dtype}


# ── inputs ───────────────────────────────────────────────────────────────────

def _spread(lo, hi, n, turn):
    """n lengths from lo to hi, spread over their logarithm, in no order."""
    if n == 1 or lo == hi:
        return [hi] * n
    return [int(round(max(lo, 1) * (hi / max(lo, 1)) ** ((turn + i * 0.6180339887) % 1.0))) for i in range(n)]


def _lengths(case):
    """(past, new) of every row; with ``idle`` = k every k-th row has no token in the step."""
    n, idle = case["seqs"], case.get("idle", 0)
    past = _spread(case["past_lo"], case["past_hi"], n, 0.999)
    if case["op"] == "read":
        return past, [0] * n
    new = _spread(case["new_lo"], case["new_hi"], n, 0.2)
    if idle and n > 1:
        new = [0 if i % idle == idle - 1 else t for i, t in enumerate(new)]
    return past, new


def _ends(case):
    """(first, count) of what a read takes of every row: its last positions."""
    past, _ = _lengths(case)
    count = [min(c, p) for c, p in zip(_spread(case["count_lo"], case["count_hi"], case["seqs"], 0.4), past)]
    return [p - c for p, c in zip(past, count)], count


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _values(g, tokens, heads, dtype):
    """Keys and values as projections leave them: each head and channel its own spread, a few channels large."""
    spread = torch.exp(0.7 * torch.randn((heads, HEAD), generator=g, device="cuda"))
    return (torch.randn((tokens, heads, HEAD), generator=g, device="cuda") * spread).to(dtype)


def _inputs(case, seed):
    """What both sides and the 64-bit results start from."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    past, new = _lengths(case)
    dtype, n_kv = DTYPES[case["dtype"]], case["n_kv"]
    total = [_pages(a + b) for a, b in zip(past, new)]
    d = {"past": past, "new": new, "width": max(_pages(max(past) + max(new)), 1), "n_pages": sum(total) + 3,
         "past_k": _values(g, sum(past), n_kv, dtype), "past_v": _values(g, sum(past), n_kv, dtype)}
    # q, k, v as slices of one projection's output
    x = torch.cat([torch.randn((sum(new), N_Q, HEAD), generator=g, device="cuda").to(dtype),
                   _values(g, sum(new), 2 * n_kv, dtype)], dim=1)
    d["q"], d["k"], d["v"] = x[:, :N_Q], x[:, N_Q:N_Q + n_kv], x[:, N_Q + n_kv:]
    # a pool that has run for a while hands its pages out in no order
    d["free"] = torch.randperm(d["n_pages"], generator=g, device="cuda").to(torch.int32)
    return d


# ── states ───────────────────────────────────────────────────────────────────

def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    d = _inputs(case, seed)
    s = _own_state(case, d) if own else _plain_state(case, d)
    s |= {"case": case, "q": d["q"], "k": d["k"], "v": d["v"], "past": _ints(d["past"]), "new": _ints(d["new"])}
    if case["op"] == "read":
        first, count = _ends(case)
        s |= {"first": _ints(first), "count": _ints(count), "n_out": max(sum(count), 1)}
    return s


def _oi2():
    at = os.path.join(os.getcwd(), "hot-cold-neural-split-openinfer2_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import oi2
    return oi2


def _own_state(case, d):
    oi2 = _oi2()
    cache = oi2.PagedKVCache(1, N_Q, case["n_kv"], case["seqs"], d["width"] * PAGE, d["n_pages"], device="cuda", bits=4)
    cache.free.copy_(d["free"])
    first = cache.new_plan(max(sum(d["past"]), 1))
    cache.extend(_ints(d["past"]), first)
    if sum(d["past"]):
        cache.append(0, d["past_k"], d["past_v"], first)
    s = {"cache": cache, "n_tokens": max(sum(d["new"]), 1)}
    if case["op"] == "read":
        return s
    s["plan"] = cache.new_plan(s["n_tokens"], max_new=max(max(d["new"]), 1))
    cache.extend(_ints(d["new"]), s["plan"])
    if case["op"] == "attend":
        cache.append(0, d["k"], d["v"], s["plan"])
    elif case["rotate"] != "none":
        s["rotary"] = oi2.Rotary(HEAD, THETA, rotary_dim=case["part"], layout=case["rotate"], device="cuda")
    return s


def _plain_state(case, d):
    """A pool of pages of codes and scales, block tables, and the step's (page, place) of every token."""
    stack, table = d["free"].tolist(), [[] for _ in d["past"]]
    for grow in (d["past"], [a + b for a, b in zip(d["past"], d["new"])]):
        for i, n in enumerate(grow):
            while len(table[i]) < _pages(n):
                table[i].append(stack.pop())
    n_kv = case["n_kv"]
    s = {"table": _ints([t + [0] * (d["width"] - len(t)) for t in table]).long(),
         "codes": [torch.zeros((d["n_pages"], PAGE, n_kv, HEAD), dtype=torch.int8, device="cuda") for _ in range(2)],
         "scales": [torch.zeros((d["n_pages"], PAGE, n_kv, HEAD // GROUP), device="cuda") for _ in range(2)],
         "width": d["width"], "max_new": max(max(d["new"]), 1)}
    past, new = _ints(d["past"]).long(), _ints(d["new"]).long()
    if sum(d["past"]):
        row, pos = _plain_rows(torch.zeros_like(past), past, sum(d["past"]))
        _plain_store(s, row, pos, d["past_k"], d["past_v"])
    if sum(d["new"]):
        s["row"], s["pos"] = _plain_rows(past, new, sum(d["new"]))
        if case["op"] == "attend":
            _plain_store(s, s["row"], s["pos"], d["k"], d["v"])
    return s


# ── one pass ─────────────────────────────────────────────────────────────────

def run(s):
    op = s["case"]["op"]
    if own:
        return {"store": _own_store, "read": _own_read, "attend": _own_attend}[op](s)
    return {"store": _plain_append, "read": _plain_read, "attend": _plain_attend}[op](s)


def _own_store(s):
    cache, q = s["cache"], None
    if "rotary" in s:
        q = cache.append(0, s["k"], s["v"], s["plan"], q=s["q"], rotary=s["rotary"])
    else:
        cache.append(0, s["k"], s["v"], s["plan"])
    k, v, _ = cache.fetch(0, s["new"], s["n_tokens"], first=s["past"], dtype=s["k"].dtype)
    return {"k": k, "v": v} if q is None else {"k": k, "v": v, "q": q}


def _own_read(s):
    k, v, cu = s["cache"].fetch(0, s["count"], s["n_out"], first=s["first"], dtype=DTYPES[s["case"]["dtype"]])
    return {"k": k, "v": v, "cu": cu}


def _own_attend(s):
    return {"out": s["cache"].attend(0, s["q"], s["plan"])}


# ── the plain forms ──────────────────────────────────────────────────────────

def _plain_rows(first, count, n):
    """Row and position of each of n packed tokens: count[i] of row i from first[i] on."""
    end = count.cumsum(0)
    t = torch.arange(n, device="cuda")
    row = torch.searchsorted(end, t, right=True)
    return row, first[row] + t - (end - count)[row]


def _plain_code(x):
    """Codes and scales of x (tokens, heads, 128)."""
    x = x.float().unflatten(-1, (HEAD // GROUP, GROUP))
    top = x.abs().amax(-1)
    y = top / TOP_CODE
    unit = torch.ldexp(torch.ones_like(y), torch.clamp(torch.frexp(y)[1] - 8, min=-24))    # 8 significant bits
    scale = (torch.round(y / unit) * unit).clamp(LEAST_SCALE, TOP_SCALE)
    scale = torch.where(top > 0, scale, 0.0)
    codes = torch.round(x / torch.where(top > 0, scale, 1.0)[..., None]).clamp(-TOP_CODE, TOP_CODE)
    return codes.to(torch.int8).flatten(-2), scale


def _plain_store(s, row, pos, k, v):
    page = s["table"][row, pos.div(PAGE, rounding_mode="floor")]
    for i, x in enumerate((k, v)):
        codes, scale = _plain_code(x)
        s["codes"][i][page, pos % PAGE] = codes
        s["scales"][i][page, pos % PAGE] = scale


def _plain_held(s, row, pos):
    """What the cache stands for at those positions, in 32 bits: k and v (tokens, heads, 128)."""
    page = s["table"][row, pos.div(PAGE, rounding_mode="floor")]
    return [(c[page, pos % PAGE].float().unflatten(-1, (HEAD // GROUP, GROUP)) * z[page, pos % PAGE][..., None]).flatten(-2)
            for c, z in zip(s["codes"], s["scales"])]


def _plain_turn(x, pos, case):
    """x (tokens, heads, 128) rotated: in 64 bits, rounded to 32 and then to its type."""
    part, half = case["part"], case["rotate"] == "half"
    f = THETA ** (-torch.arange(part // 2, dtype=torch.float64, device="cuda") * 2 / part)
    angle = pos.double()[:, None, None] * f
    y = x.double()
    a, b = (y[..., :part // 2], y[..., part // 2:part]) if half else (y[..., 0:part:2], y[..., 1:part:2])
    c, d = a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()
    z = torch.cat([c, d], -1) if half else torch.stack([c, d], -1).flatten(-2)
    return torch.cat([z, y[..., part:]], -1).float().to(x.dtype)


def _plain_append(s):
    case, k, out = s["case"], s["k"], {}
    if case["rotate"] != "none":
        q, k = (_plain_turn(x, s["pos"], case) for x in (s["q"], k))
        out = {"q": q}
    _plain_store(s, s["row"], s["pos"], k, s["v"])
    k, v = (x.to(s["k"].dtype) for x in _plain_held(s, s["row"], s["pos"]))
    return {"k": k, "v": v, **out}


def _plain_read(s):
    count = s["count"].long()
    row, pos = _plain_rows(s["first"].long(), count, s["n_out"])
    k, v = (x.to(DTYPES[s["case"]["dtype"]]) for x in _plain_held(s, row, pos))
    return {"k": k, "v": v, "cu": torch.cat([torch.zeros_like(count[:1]), count.cumsum(0)]).int()}


def _plain_attend(s):
    case, n, n_kv, m, width = s["case"], s["case"]["seqs"], s["case"]["n_kv"], s["max_new"], s["width"]

    def rows(i):                                   # (rows, heads, width * 64, 128)
        x = s["codes"][i][s["table"]].float().unflatten(-1, (HEAD // GROUP, GROUP)) * s["scales"][i][s["table"]][..., None]
        return x.flatten(-2).flatten(1, 2).transpose(1, 2)

    # the packed query tokens as (rows, most tokens of a row)
    t = torch.arange(m, device="cuda")
    new, past = s["new"].long(), s["past"].long()
    real = t < new[:, None]
    index = torch.where(real, (new.cumsum(0) - new)[:, None] + t, 0)
    q = s["q"].float()[index].reshape(n, m, n_kv, N_Q // n_kv, HEAD).permute(0, 2, 3, 1, 4).reshape(n, n_kv, -1, HEAD)
    pos = torch.arange(width * PAGE, device="cuda")
    seen = real[..., None] & (pos <= past[:, None, None] + t[:, None])
    score = torch.matmul(q * HEAD ** -0.5, rows(0).transpose(2, 3)).reshape(n, N_Q, m, -1)
    score = torch.where(seen[:, None], score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.reshape(n, n_kv, -1, width * PAGE), rows(1)).reshape(n, N_Q, m, HEAD)
    out = torch.where(total > 0, out / total, 0.0).transpose(1, 2)
    y = torch.empty(s["q"].shape, dtype=s["q"].dtype, device="cuda")
    y[index[real]] = out[real].to(y.dtype)
    return {"out": y}


# ── least work ───────────────────────────────────────────────────────────────

def work(case):
    n_kv = case["n_kv"]
    held = 2 * n_kv * (HEAD // 2 + HEAD // GROUP * 2)       # bytes of a position's k and v in the cache
    dense = 2 * n_kv * HEAD * 2                             # ... and as values of 16 bits
    if case["op"] == "read":
        tokens = sum(_ends(case)[1])
        return {"bytes": tokens * (held + dense) + 12 * case["seqs"], "flops": tokens * dense // 2}
    past, new = _lengths(case)
    tokens = sum(new)
    if case["op"] == "store":
        turned = tokens * (N_Q + n_kv) * case["part"]
        q = 2 * tokens * N_Q * HEAD * 2 if turned else 0
        # values in; codes out, and in again; values out
        return {"bytes": 2 * tokens * (dense + held) + q, "flops": 3 * turned + 4 * tokens * dense // 2}
    read = sum(a + b for a, b in zip(past, new) if b)
    pairs = sum(b * a + b * (b + 1) // 2 for a, b in zip(past, new))
    return {"bytes": read * held + 2 * tokens * N_Q * HEAD * 2, "flops": 4 * pairs * N_Q * HEAD}


# ── results in 64 bits, from the definitions ─────────────────────────────────

def _coded64(x):
    """What x (tokens, heads, 128) stands for once coded, group by group."""
    parts = []
    for c in range(HEAD // GROUP):
        g = x[..., GROUP * c:GROUP * (c + 1)].double()
        top = torch.maximum(g.amax(-1, keepdim=True), -g.amin(-1, keepdim=True))
        step = torch.exp2(torch.clamp(torch.floor(torch.log2((top / 7).clamp(min=1e-30))) - 7, min=-24.0).round())
        scale = torch.round(top / 7 / step) * step          # halves to even
        scale = torch.minimum(torch.maximum(scale, torch.full_like(scale, 2.0 ** -24)), torch.full_like(scale, 9344.0))
        codes = torch.minimum(torch.round(g.abs() / scale), torch.full_like(g, 7.0)) * torch.sign(g)
        parts.append(torch.where(top > 0, codes * scale, torch.zeros_like(g)))
    return torch.cat(parts, -1)


def _turn64(x, positions, case):
    part, y = case["part"], x.double().clone()
    for i in range(part // 2):
        a, b = (i, i + part // 2) if case["rotate"] == "half" else (2 * i, 2 * i + 1)
        angle = positions.double() * THETA ** (-2.0 * i / part)
        z = torch.complex(x[..., a].double(), x[..., b].double()) * torch.polar(torch.ones_like(angle), angle)[:, None]
        y[..., a], y[..., b] = z.real, z.imag
    return y


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "read":
        first, count = _ends(case)
        at, t0 = [], 0
        for p, f, c in zip(d["past"], first, count):
            at.append(torch.arange(t0 + f, t0 + f + c, device="cuda"))
            t0 += p
        at = torch.cat(at)
        return {"k": _coded64(d["past_k"][at]), "v": _coded64(d["past_v"][at]), "cu": None}
    if case["op"] == "store":
        if case["rotate"] == "none":
            return {"k": _coded64(d["k"]), "v": _coded64(d["v"])}
        pos = torch.tensor([a + t for a, b in zip(d["past"], d["new"]) for t in range(b)], device="cuda")
        # a key is rounded to its type before it is coded
        k = _turn64(d["k"], pos, case).to(d["k"].dtype)
        return {"k": _coded64(k), "v": _coded64(d["v"]), "q": _turn64(d["q"], pos, case)}
    group, out, t0, t1 = N_Q // case["n_kv"], [], 0, 0
    for a, b in zip(d["past"], d["new"]):
        x = [_coded64(torch.cat([d["past_" + c][t0:t0 + a], d[c][t1:t1 + b]])) if b else None for c in "kv"]
        q = d["q"][t1:t1 + b].double()
        t0, t1 = t0 + a, t1 + b
        if not b:
            continue
        heads = []
        for h in range(N_Q):
            z = q[:, h] @ x[0][:, h // group].T / math.sqrt(HEAD)
            z = z.masked_fill(torch.arange(a + b, device="cuda") > a + torch.arange(b, device="cuda")[:, None], -math.inf)
            heads.append(torch.softmax(z, -1) @ x[1][:, h // group])
        out.append(torch.stack(heads, 1))
    return {"out": torch.cat(out)}
