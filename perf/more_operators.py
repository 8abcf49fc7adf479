"""The index branch of a sparse attention step, case by case: what finds the cached rows that the
sparse attention reads.

- ``write``   index queries and keys rotated, quantized to FP8, and the keys written to their paged
              cache (``ops.IndexWrite``).
- ``scores``  a cheap score of every cached row for every query token (``ops.IndexScores``).
- ``select``  the best rows, or the best pages of 64 rows, of each token (``ops.IndexSelect``).

``run`` computes them with elementary torch operations in 32 bits, or, where ``own`` is true, with
this framework's kernels. ``exact`` gives the definition's values in 64 bits.
"""

import math
import os
import sys

import torch

own = False

PAGE = 64
DIM = 128  # width of an index query and of an index key
ROW = 144  # bytes of an index cache row: 128 codes, a 32-bit scale, padding
EPS = 1e-6


def listed():
    return [
        # One token of one request: latency. Rotary part in front of the head, interleaved pairs.
        {"name": "write-one-token", "op": "write", "heads": 64, "new": "1", "requests": 1, "longest": 8192, "rope": 64, "start": 0, "half": False, "norm": "layer"},
        # A decode batch, no rotary part (the model without positions in its cache).
        {"name": "write-decode-64", "op": "write", "heads": 32, "new": "1", "requests": 64, "longest": 32768, "rope": 0, "start": 0, "half": False, "norm": "rms"},
        # A prefill step: the halves of the rotary part turned against each other.
        {"name": "write-prefill-8k", "op": "write", "heads": 64, "new": "8192", "requests": 1, "longest": 8192, "rope": 64, "start": 0, "half": True, "norm": "layer"},
        # Odd chunks at far positions, the rotary part at the end of the head.
        {"name": "write-ragged-far", "op": "write", "heads": 48, "new": "333,1,77,610", "requests": 4, "longest": 131072, "rope": 32, "start": 96, "half": False, "norm": "none"},
        # One request alone: latency.
        {"name": "scores-one-8k", "op": "scores", "heads": 64, "new": "1", "requests": 1, "longest": 8192},
        # A decode batch over long contexts.
        {"name": "scores-decode-64", "op": "scores", "heads": 64, "new": "1", "requests": 64, "longest": 32768},
        # Two to four tokens a request, odd lengths, a head count that is no power of two.
        {"name": "scores-drafts-ragged", "op": "scores", "heads": 48, "new": "2,4,1,3,2", "requests": 45, "longest": 10007},
        # Chunked prefill over a cached prefix.
        {"name": "scores-prefill-2k", "op": "scores", "heads": 64, "new": "2048", "requests": 1, "longest": 8192},
        # One row: latency.
        {"name": "select-one-8k", "op": "select", "new": "1", "requests": 1, "longest": 8192, "k": 2048, "pages": False, "values": "f32"},
        # A decode batch, the sparse benchmark's sizes.
        {"name": "select-decode-64", "op": "select", "new": "1", "requests": 64, "longest": 32768, "k": 2048, "pages": False, "values": "f32"},
        # A prefill step: from tokens that see less than k rows to tokens that see them all.
        {"name": "select-prefill-2k", "op": "select", "new": "2048", "requests": 1, "longest": 16384, "k": 2048, "pages": False, "values": "f32"},
        # Pages of long contexts for a decode batch, first and last page kept.
        {"name": "select-pages-64", "op": "select", "new": "1", "requests": 64, "longest": 131072, "k": 64, "pages": True, "values": "f32"},
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["write", "scores", "select"])
    requests = _spread(rng, 1, 64)
    new = [1] if rng.random() < 0.4 else [_spread(rng, 1, max(1, 2048 // requests)) for _ in range(min(requests, rng.randint(1, 4)))]
    case = {"op": op, "new": ",".join(map(str, new)), "requests": requests}
    if op == "write":
        rope = rng.choice([0, 16, 32, 64, 128])
        case.update(heads=16 * rng.randint(1, 8), longest=max(max(new), _spread(rng, 1, 2 ** 20 // requests)), rope=rope,
                    start=rng.choice([0, DIM - rope]), half=rng.random() < 0.5, norm=rng.choice(["none", "rms", "layer"]))
    elif op == "scores":
        heads = 16 * rng.randint(1, 8)
        # the plain form pads: its scores stay within the largest listed cases'
        most = 2 ** 30 // (heads * requests * max(new))
        case.update(heads=heads, longest=max(max(new), _spread(rng, 64, min(32768, max(64, most)))))
    else:
        pages = rng.random() < 0.35
        tokens = sum(new[i % len(new)] for i in range(requests))
        case.update(longest=max(max(new), _spread(rng, 64, min(131072, 2 ** 23 // tokens + 64))), k=_spread(rng, 1, 200 if pages else 2051),
                    pages=pages, values=rng.choice(["f32", "f32", "bf16"]))
    return case


# ------------------------------------------------------------------------------------- inputs


def _ops():
    """The framework's operators, reached as a user reaches them."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "tensorquay-engine_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from tq_mla import ops
    return ops


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _batch(case):
    """New tokens and cached rows (the new ones among them) of each request. Lengths fall from the
    longest to half of it."""
    each = [int(x) for x in case["new"].split(",")]
    new = [each[i % len(each)] for i in range(case["requests"])]
    span = max(1, case["longest"] // 2)
    lens = [max(n, case["longest"] - (i * 977) % span) for i, n in enumerate(new)]
    return new, lens


def _tokens(case):
    new, lens = _batch(case)
    n, c = torch.tensor(new, device="cuda"), torch.tensor(lens, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), n)
    first = torch.cumsum(n, 0) - n
    pos = torch.arange(len(seq), device="cuda") - first[seq] + (c - n)[seq]
    return {"seq_id": seq.to(torch.int32), "q_pos": pos.to(torch.int32), "kv_len": c.to(torch.int32), "first": first}


def _pages(g, lens):
    """A page table in no order; entries past a request's pages are empty."""
    need = torch.tensor([-(-n // PAGE) for n in lens], device="cuda")
    total, slots = int(need.sum()), int(need.max())
    order = torch.randperm(total + 3, generator=g, device="cuda").to(torch.int32)
    held = torch.arange(slots, device="cuda")[None] < need[:, None]
    table = torch.full((len(lens), slots), -1, dtype=torch.int32, device="cuda")
    table[held] = order[:total]
    return table, total + 3


def _quantize(x):
    """Rows of 128 values as E4M3 codes and a scale a row (a row of zeros: scale 0, codes 0)."""
    peak = x.abs().amax(dim=-1, keepdim=True)
    codes = (x * torch.where(peak > 0, 448.0 / peak, 0.0)).to(torch.float8_e4m3fn)
    return codes, peak[..., 0] / 448.0


def _codes(kv):
    return kv[..., :DIM].view(torch.float8_e4m3fn)


def _scales(kv):
    return kv.view(torch.float32)[..., DIM // 4]


def _prepare_write(case, seed):
    g = _generator(seed)
    st = {"op": "write", "case": case, **_tokens(case)}
    _, lens = _batch(case)
    t, h = st["seq_id"].numel(), case["heads"]
    st["page_table"], pages = _pages(g, lens)
    st["kv"] = torch.zeros((pages, PAGE, ROW), dtype=torch.uint8, device="cuda")
    st["q"] = (2.0 * _normal(g, t, h, DIM)).to(torch.bfloat16)
    st["k"] = (1.5 * _normal(g, t, DIM) + 0.3).to(torch.bfloat16)
    st["w"] = _normal(g, t, h).to(torch.bfloat16)
    st["scale"] = h ** -0.5 * DIM ** -0.5
    st["norm_weight"] = (1.0 + 0.2 * _normal(g, DIM)).to(torch.bfloat16) if case["norm"] != "none" else None
    st["norm_bias"] = (0.1 * _normal(g, DIM)).to(torch.bfloat16) if case["norm"] == "layer" else None
    st["freq"], st["mscale"] = None, 1.0
    if case["rope"]:
        # base 10000, positions stretched four times for long contexts
        at = torch.arange(0, case["rope"], 2, device="cuda", dtype=torch.float64) / case["rope"]
        st["freq"] = (10000.0 ** -at / 4.0).float()
        st["mscale"] = 0.1 * math.log(4.0) + 1.0
    if own:
        st["codes"] = torch.empty((t, h, DIM), dtype=torch.uint8, device="cuda")
        st["weights"] = torch.empty((t, h), dtype=torch.float32, device="cuda")
        st["launch"] = _ops().IndexWrite(
            st["q"], st["k"], st["w"], st["page_table"], st["seq_id"], st["q_pos"], st["kv"], st["codes"], st["weights"],
            scale=st["scale"], norm_weight=st["norm_weight"], norm_bias=st["norm_bias"], eps=EPS, freq=st["freq"],
            rope_start=case["start"], rope_half=case["half"], rope_mscale=st["mscale"])
    return st


def _prepare_scores(case, seed):
    g = _generator(seed)
    st = {"op": "scores", "case": case, **_tokens(case)}
    _, lens = _batch(case)
    t, h = st["seq_id"].numel(), case["heads"]
    st["page_table"], pages = _pages(g, lens)
    # rows of earlier requests fill what no request holds
    codes, scale = _quantize(1.5 * _normal(g, pages * PAGE, DIM))
    kv = torch.zeros((pages * PAGE, ROW), dtype=torch.uint8, device="cuda")
    kv[:, :DIM] = codes.view(torch.uint8)
    kv.view(torch.float32)[:, DIM // 4] = scale
    st["kv"] = kv.view(pages, PAGE, ROW)
    codes, scale = _quantize(2.0 * _normal(g, t, h, DIM))
    st["q"] = codes.view(torch.uint8)
    st["w"] = _normal(g, t, h) * scale * (h * DIM) ** -0.5
    # columns behind a token's last visible row keep what they hold
    st["scores"] = torch.zeros((t, -(-case["longest"] // PAGE) * PAGE), dtype=torch.float32, device="cuda")
    if own:
        st["launch"] = _ops().IndexScores(st["q"], st["w"], st["kv"], st["page_table"], st["seq_id"], st["q_pos"], st["kv_len"], st["scores"])
    return st


def _prepare_select(case, seed):
    g = _generator(seed)
    st = {"op": "select", "case": case, **_tokens(case)}
    _, lens = _batch(case)
    t = st["seq_id"].numel()
    st["page_table"], _ = _pages(g, lens)
    # weighted sums over heads of what is positive, a few rows of each context far above the others
    width = -(-case["longest"] // PAGE) * PAGE
    scores = torch.einsum("tj,tjn->tn", _normal(g, t, 4), _normal(g, t, 4, width).relu_())
    scores += 2.0 * torch.rand((t, width), generator=g, device="cuda").pow_(8)
    if case["values"] == "bf16":  # scores that were kept in 16 bits: many are equal
        scores = scores.to(torch.bfloat16).float()
    st["scores"] = scores
    st["keep"] = 1 if case["pages"] else 0
    if own:
        st["idx"] = torch.empty((t, case["k"]), dtype=torch.int32, device="cuda")
        st["len"] = torch.empty((t,), dtype=torch.int32, device="cuda")
        st["launch"] = _ops().IndexSelect(
            scores, st["seq_id"], st["q_pos"], st["kv_len"], st["idx"], st["len"], page_table=st["page_table"] if case["pages"] else None,
            keep_first=st["keep"], keep_last=st["keep"])
    return st


def prepare(case, seed):
    return {"write": _prepare_write, "scores": _prepare_scores, "select": _prepare_select}[case["op"]](case, seed)


# ------------------------------------------------------------------------------------- plain forms


def _turned(st, x):
    """Rows ``[T, ..., 128]`` with their rotary part turned by their token's position."""
    case = st["case"]
    if not case["rope"]:
        return x
    lo, hi = case["start"], case["start"] + case["rope"]
    angle = st["q_pos"].double()[:, None] * st["freq"].double()
    shape = (len(angle),) + (1,) * (x.dim() - 2) + (-1,)
    cos, sin = (angle.cos() * st["mscale"]).float().view(shape), (angle.sin() * st["mscale"]).float().view(shape)
    part = x[..., lo:hi]
    if case["half"]:
        a, b = part.chunk(2, dim=-1)
        part = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    return torch.cat([x[..., :lo], part, x[..., hi:]], dim=-1)


def _plain_write(st):
    k = st["k"].float()
    if st["norm_weight"] is not None:
        if st["norm_bias"] is not None:
            k = k - k.mean(dim=1, keepdim=True)
        k = k * torch.rsqrt((k * k).mean(dim=1, keepdim=True) + EPS) * st["norm_weight"].float()
        if st["norm_bias"] is not None:
            k = k + st["norm_bias"].float()
    codes, scale = _quantize(_turned(st, k))
    page = st["page_table"][st["seq_id"].long(), st["q_pos"].long() // PAGE].long()
    row = page * PAGE + st["q_pos"].long() % PAGE
    _codes(st["kv"]).view(torch.uint8).view(-1, DIM)[row] = codes.view(torch.uint8)
    _scales(st["kv"]).view(-1)[row] = scale
    codes, scale = _quantize(_turned(st, st["q"].float()))
    return {"q": codes, "w": st["w"].float() * st["scale"] * scale, "keys": _codes(st["kv"]), "key_scale": _scales(st["kv"])}


def _plain_scores(st):
    new, lens = _batch(st["case"])
    keys, longest = max(lens), max(new)
    pos = torch.arange(keys, device="cuda")
    page = st["page_table"].long().clamp_min(0)[:, pos // PAGE] * PAGE + pos % PAGE
    k = _codes(st["kv"]).reshape(-1, DIM)[page].float()
    k_scale = _scales(st["kv"]).reshape(-1)[page]
    # the batch padded to its most new tokens and its longest cache
    seq, first = st["seq_id"].long(), st["first"]
    last = torch.tensor(new, device="cuda") - 1
    token = first[:, None] + torch.minimum(torch.arange(longest, device="cuda")[None], last[:, None])
    q = st["q"].view(torch.float8_e4m3fn)[token].float()
    s, t, h, _ = q.shape
    dots = torch.bmm(q.view(s, t * h, DIM), k.transpose(1, 2)).relu_()
    got = torch.bmm(st["w"][token].view(s * t, 1, h), dots.view(s * t, h, keys)).view(s, t, keys) * k_scale[:, None]
    sees = torch.minimum(st["kv_len"].long()[seq], st["q_pos"].long() + 1)
    at = torch.arange(len(seq), device="cuda") - first[seq]
    st["scores"][:, :keys] = torch.where(pos[None] < sees[:, None], got[seq, at], st["scores"][:, :keys])
    return {"scores": st["scores"]}


def _plain_select(st):
    case, scores, k = st["case"], st["scores"], st["case"]["k"]
    seq = st["seq_id"].long()
    sees = torch.minimum(st["kv_len"].long()[seq], st["q_pos"].long() + 1)
    column = torch.arange(scores.shape[1], device="cuda")
    value = torch.where(column[None] < sees[:, None], scores, -math.inf)
    value = torch.where(torch.isnan(value), -math.inf, value)
    count = sees
    if case["pages"]:
        value = value.view(len(seq), -1, PAGE).amax(dim=2)
        count = (sees + PAGE - 1) // PAGE
        column = torch.arange(value.shape[1], device="cuda")
        kept = (column[None] < st["keep"]) | (column[None] >= count[:, None] - st["keep"])
        value = torch.where(kept & (column[None] < count[:, None]), math.inf, value)
    best, at = torch.sort(value, dim=1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    taken = (best > -math.inf).sum(dim=1)
    far = scores.shape[1]
    at = torch.sort(torch.where(best > -math.inf, at, far), dim=1)[0]
    at = torch.nn.functional.pad(at, (0, k - at.shape[1]), value=far)
    held = at < far
    if not case["pages"]:
        return {"idx": torch.where(held, at, -1).to(torch.int32), "len": taken.to(torch.int32)}
    table = st["page_table"][seq[:, None], at.clamp_max(st["page_table"].shape[1] - 1)]
    ends = (held & (at == count[:, None] - 1)).any(dim=1)
    rows = taken * PAGE - torch.where(ends, count * PAGE - sees, 0)
    return {"idx": torch.where(held, table, -1).to(torch.int32), "len": rows.to(torch.int32)}


def run(state):
    op = state["op"]
    if not own:
        return {"write": _plain_write, "scores": _plain_scores, "select": _plain_select}[op](state)
    state["launch"]()
    if op == "write":
        return {"q": state["codes"].view(torch.float8_e4m3fn), "w": state["weights"], "keys": _codes(state["kv"]), "key_scale": _scales(state["kv"])}
    if op == "scores":
        return {"scores": state["scores"]}
    return {"idx": state["idx"], "len": state["len"]}


# ------------------------------------------------------------------------------------- definition in 64 bits


def _grid(x):
    """The nearest E4M3 values, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _exact_rows(st, x):
    """Rotary part as complex numbers, then codes and scale."""
    case = st["case"]
    if case["rope"]:
        lo, n = case["start"], case["rope"] // 2
        i = torch.arange(n, device="cuda")
        re, im = (lo + i, lo + i + n) if case["half"] else (lo + 2 * i, lo + 2 * i + 1)
        turn = torch.polar(torch.full((len(x), n), st["mscale"], dtype=torch.float64, device="cuda"), st["q_pos"].double()[:, None] * st["freq"].double())
        z = torch.complex(x[..., re], x[..., im]) * (turn if x.dim() == 2 else turn[:, None])
        x = x.clone()
        x[..., re], x[..., im] = z.real, z.imag
    scale = x.abs().amax(dim=-1) / 448.0
    return _grid(x / torch.where(scale > 0, scale, 1.0)[..., None]), scale


def _exact_write(case, seed):
    st = _prepare_write(case, seed)
    k = st["k"].double()
    if case["norm"] == "rms":
        k = k / (k.square().sum(1, keepdim=True) / DIM + EPS).sqrt() * st["norm_weight"].double()
    if case["norm"] == "layer":
        k = (k - k.sum(1, keepdim=True) / DIM) / (k.var(1, unbiased=False, keepdim=True) + EPS).sqrt()
        k = k * st["norm_weight"].double() + st["norm_bias"].double()
    codes, scale = _exact_rows(st, k)
    keys = torch.zeros((st["kv"].shape[0], PAGE, DIM), dtype=torch.float64, device="cuda")
    key_scale = torch.zeros(keys.shape[:2], dtype=torch.float64, device="cuda")
    pos = st["q_pos"].long()
    page = st["page_table"][st["seq_id"].long(), pos // PAGE].long()
    keys[page, pos % PAGE], key_scale[page, pos % PAGE] = codes, scale
    codes, scale = _exact_rows(st, st["q"].double())
    return {"q": codes, "w": st["w"].double() * st["scale"] * scale, "keys": keys, "key_scale": key_scale}


def _exact_scores(case, seed):
    """Request by request and head by head."""
    st = _prepare_scores(case, seed)
    new, lens = _batch(case)
    scores = torch.zeros(st["scores"].shape, dtype=torch.float64, device="cuda")
    start = 0
    for s, (n, c) in enumerate(zip(new, lens)):
        pages = st["kv"][st["page_table"][s, :-(-c // PAGE)].long()]
        k = (_codes(pages).double() * _scales(pages).double()[..., None]).view(-1, DIM)[:c]
        q = st["q"][start:start + n].view(torch.float8_e4m3fn).double()
        for h in range(case["heads"]):
            scores[start:start + n, :c] += st["w"][start:start + n, h, None].double() * torch.clamp(q[:, h] @ k.T, min=0.0)
        start += n
    pos = torch.arange(scores.shape[1], device="cuda")
    return {"scores": scores.masked_fill_(pos[None] > st["q_pos"][:, None], 0.0)}


def exact(case, seed):
    """What is selected is whole numbers: they are compared as they are."""
    if case["op"] == "write":
        return _exact_write(case, seed)
    return _exact_scores(case, seed) if case["op"] == "scores" else None


# ------------------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    new, lens = _batch(case)
    tokens = sum(new)
    sees = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(new, lens))
    if case["op"] == "write":
        h = case["heads"]
        return {"bytes": tokens * (h * (3 * DIM + 6) + 3 * DIM + 16), "flops": tokens * (h + 1) * DIM * 6}
    if case["op"] == "scores":
        h = case["heads"]
        return {"bytes": sum(lens) * (DIM + 4) + tokens * h * (DIM + 4) + 4 * sees, "flops": sees * h * 2 * (DIM + 1)}
    return {"bytes": 4 * sees + 4 * tokens * case["k"], "flops": sees}
