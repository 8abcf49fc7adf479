"""The operators around a chunk of new tokens, case by case: what a serving step over the paged
latent cache runs beside the projections.

- ``plan``   the step's metadata from its request lengths (``ops.StepPlan``): which sequence,
             position and pool row each new token has, and the pages that the cache grows by.
- ``chunk``  attention of each request's chunk of new tokens over its paged latent rows, with
             per-head keys and values expanded from them (``ops.MlaChunk``).
- ``norm``   the block's output norm, gate and scaled residual sum, and the norm before the next
             block, in one pass (``ops.BlockNorm``).

``run`` computes them with elementary torch operations in 32 bits, or, where ``own`` is true, with
this framework's kernels. ``exact`` gives the definition's values in 64 bits.
"""

import math
import os
import sys

import torch

own = False

PAGE = 64
LATENT = 512
EPS = 1e-6
#: Row formats by name: format code, RoPE width, key width without RoPE, value width, row bytes.
FORMATS = {"bf16": (0, 0, 256, 256, 1024), "fp8": (1, 0, 256, 256, 544), "rope": (2, 64, 128, 128, 1152)}


def listed():
    return [
        # A short follow-up question on a short conversation: latency, one tensor-parallel shard.
        {"name": "chunk-short", "op": "chunk", "rows": "rope", "heads": 16, "new": "24", "cached": "100"},
        # Chunked prefill of two long prompts, all heads on one GPU: the prefill benchmark's shape.
        {"name": "chunk-2k-prefix", "op": "chunk", "rows": "rope", "heads": 128, "new": "2048,2048", "cached": "6144,2500"},
        # First chunk of one prompt: nothing cached before it, 256-wide heads.
        {"name": "chunk-first-4k", "op": "chunk", "rows": "bf16", "heads": 64, "new": "4096", "cached": "0"},
        # A mixed step over FP8 rows: odd chunks, a single token, an empty prefix.
        {"name": "chunk-fp8-ragged", "op": "chunk", "rows": "fp8", "heads": 64, "new": "333,1,1023,77,640", "cached": "1000,4001,0,2047,3001"},
        # The last few tokens of a long document: few query rows, a long cache.
        {"name": "chunk-long-tail", "op": "chunk", "rows": "rope", "heads": 32, "new": "192", "cached": "65300"},
        # One token's residual step between two blocks.
        {"name": "norm-one-token", "op": "norm", "tokens": 1, "width": 7168, "residual": "bf16", "post": False, "gate": "none", "pre": True},
        # A decode batch with norms on both sides of the block and a gate per channel.
        {"name": "norm-decode-64", "op": "norm", "tokens": 64, "width": 4096, "residual": "bf16", "post": True, "gate": "channel", "pre": True},
        # A prefill step: the residual stream kept in 32 bits, a gate per token and channel.
        {"name": "norm-prefill-8k", "op": "norm", "tokens": 8192, "width": 7168, "residual": "f32", "post": True, "gate": "token", "pre": True},
        # The sum alone after the last block, an odd number of rows of an odd width.
        {"name": "norm-odd-sum", "op": "norm", "tokens": 1021, "width": 5192, "residual": "bf16", "post": True, "gate": "none", "pre": False},
        # A decode step of a full batch.
        {"name": "plan-decode-64", "op": "plan", "requests": 64, "chunks": 0, "chunk": 1, "cached": 8192, "padding": 0},
        # Decode requests and a few prompt chunks in one step, padded to a captured batch size.
        {"name": "plan-mixed-512", "op": "plan", "requests": 512, "chunks": 7, "chunk": 2048, "cached": 65536, "padding": 211},
        # Thousands of short requests that begin together.
        {"name": "plan-burst-4k", "op": "plan", "requests": 4096, "chunks": 4000, "chunk": 97, "cached": 1024, "padding": 1000},
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "norm", "plan"])
    if op == "chunk":
        heads = rng.choice([8, 16, 32, 64, 128])
        rows = rng.choice(["rope", "bf16", "fp8"])
        seqs = rng.randint(1, 5)
        new = [_spread(rng, 1, 2048) for _ in range(seqs)]
        cached = [0 if rng.random() < 0.2 else _spread(rng, 1, 6144) for _ in range(seqs)]
        # the plain form pads: its scores stay within the largest listed case's
        while len(new) > 1 and heads * len(new) * max(new) * max(n + c for n, c in zip(new, cached)) > 2 ** 31:
            new.pop()
            cached.pop()
        return {"op": op, "rows": rows, "heads": heads, "new": ",".join(map(str, new)), "cached": ",".join(map(str, cached))}
    if op == "norm":
        return {"op": op, "tokens": _spread(rng, 1, 8192), "width": 8 * _spread(rng, 8, 896), "residual": rng.choice(["bf16", "f32"]),
                "post": rng.random() < 0.5, "gate": rng.choice(["none", "channel", "token"]), "pre": rng.random() < 0.8}
    requests = _spread(rng, 1, 4096)
    chunks = rng.randint(0, min(requests, 200))
    return {"op": op, "requests": requests, "chunks": chunks, "chunk": _spread(rng, 1, 1500), "cached": _spread(rng, 1, 65536), "padding": rng.randint(0, 300)}


# ------------------------------------------------------------------------------------- inputs


def _ops():
    """The framework's operators, reached as a user reaches them."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "tensorquay-engine_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from tq_mla import ops
    return ops


def _ints(text):
    return [int(x) for x in text.split(",")]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _fp8_rows(x):
    """Rows of 512 values as 512 E4M3 codes and one f32 scale per 128 values, in 544 bytes."""
    tiles = x.view(-1, 4, 128)
    scale = tiles.abs().amax(dim=2) / 448.0
    codes = (tiles / scale[:, :, None]).to(torch.float8_e4m3fn).view(-1, 512).view(torch.uint8)
    rows = torch.zeros((x.shape[0], 544), dtype=torch.uint8, device=x.device)
    rows[:, :512] = codes
    rows[:, 512:528] = scale.contiguous().view(torch.uint8).view(-1, 16)
    return rows


def _prepare_chunk(case, seed):
    g = _generator(seed)
    fmt, dr, dn, dv, row_bytes = FORMATS[case["rows"]]
    heads, new, cached = case["heads"], _ints(case["new"]), _ints(case["cached"])
    lens = [n + c for n, c in zip(new, cached)]
    seqs, tokens = len(new), sum(new)
    need = [-(-n // PAGE) for n in lens]
    slots, pages = max(need), sum(need) + 3
    # pages in no order; table entries past a sequence's pages are empty
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((seqs, slots), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    # cached rows; a page's rows that hold no token hold whatever was there before
    rows = torch.cat([table[s].long().clamp_min(0).repeat_interleave(PAGE)[:n] * PAGE +
                      torch.arange(n, device="cuda") % PAGE for s, n in enumerate(lens)])
    values = _normal(g, len(rows), LATENT + dr).to(torch.bfloat16)
    if case["rows"] == "fp8":
        pool = torch.full((pages * PAGE, row_bytes), 255, dtype=torch.uint8, device="cuda")
        pool[rows] = _fp8_rows(values.float())
    else:
        pool = torch.full((pages * PAGE, LATENT + dr), math.nan, dtype=torch.bfloat16, device="cuda")
        pool[rows] = values
    pool = pool.view(pages, PAGE, -1)
    starts = [sum(new[:s]) for s in range(seqs + 1)]
    state = {
        "op": "chunk", "case": case, "fmt": fmt, "dr": dr, "dn": dn, "dv": dv, "scale": (dn + dr) ** -0.5,
        "q": _normal(g, tokens, heads, dn + dr).to(torch.bfloat16),
        "w_uk": (_normal(g, heads, dn, LATENT) * LATENT ** -0.5).to(torch.bfloat16),
        "w_uv": (_normal(g, heads, dv, LATENT) * LATENT ** -0.5).to(torch.bfloat16),
        "kv": pool, "page_table": table, "q_start": _int32(starts), "kv_len": _int32(lens),
        "q_pos": torch.cat([torch.arange(c, c + n, dtype=torch.int32, device="cuda") for n, c in zip(new, cached)]),
    }
    if own:
        state["out"] = torch.empty((tokens, heads, dv), dtype=torch.bfloat16, device="cuda")
        state["launch"] = _ops().MlaChunk(
            state["q"], state["w_uk"], state["w_uv"], state["kv"], state["page_table"], state["q_start"], state["q_pos"],
            state["kv_len"], state["out"], scale=state["scale"], kv_format=fmt, max_keys=sum(lens))
    return state


def _prepare_norm(case, seed):
    g = _generator(seed)
    t, d = case["tokens"], case["width"]
    kind = torch.float32 if case["residual"] == "f32" else torch.bfloat16
    weight = lambda: (1.0 + 0.2 * _normal(g, d)).to(torch.bfloat16)  # noqa: E731
    state = {
        "op": "norm", "case": case, "scale": 0.7,
        "y": (1.5 * _normal(g, t, d)).to(torch.bfloat16), "residual": (4.0 * _normal(g, t, d)).to(kind),
        "post": weight() if case["post"] else None, "pre": weight() if case["pre"] else None,
        "gate": None if case["gate"] == "none" else torch.sigmoid(_normal(g, *((d,) if case["gate"] == "channel" else (t, d)))).to(torch.bfloat16),
    }
    if own:
        state["out"] = torch.empty((t, d), dtype=kind, device="cuda")
        state["x"] = torch.empty((t, d), dtype=torch.bfloat16, device="cuda") if case["pre"] else None
        state["launch"] = _ops().BlockNorm(
            state["y"], state["residual"], state["out"], state["x"], post_weight=state["post"], gate=state["gate"],
            scale=state["scale"], pre_weight=state["pre"], eps=EPS)
    return state


def _prepare_plan(case, seed):
    g = _generator(seed)
    n, chunks = case["requests"], case["chunks"]
    new = torch.ones(n, dtype=torch.int32, device="cuda")
    new[torch.randperm(n, generator=g, device="cuda")[:chunks]] = case["chunk"]
    cached = torch.randint(0, case["cached"] + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
    slots = -(-(case["cached"] + case["chunk"]) // PAGE)
    order = torch.randperm(n * slots + 9, generator=g, device="cuda").to(torch.int32)
    # every request holds the pages of its cached rows; all others are free
    held = torch.arange(slots, device="cuda")[None] < ((cached + PAGE - 1) // PAGE)[:, None]
    table = torch.where(held, order[:n * slots].view(n, slots), -1).to(torch.int32)
    free = torch.cat([order[:n * slots][~held.view(-1)], order[n * slots:]])
    state = {"op": "plan", "case": case, "cached_len": cached, "new_len": new, "page_table": table, "free_pages": free,
             "free_count": _int32([free.numel()]), "tokens": n - chunks + chunks * case["chunk"] + case["padding"]}
    if own:
        state["launch"] = _ops().StepPlan(cached, new, table, free, state["free_count"], tokens=state["tokens"])
    return state


def prepare(case, seed):
    return {"chunk": _prepare_chunk, "norm": _prepare_norm, "plan": _prepare_plan}[case["op"]](case, seed)


# ------------------------------------------------------------------------------------- plain forms


def _row_values(st, rows):
    """Pool rows (any leading shape) as 32-bit values."""
    flat = st["kv"].view(-1, st["kv"].shape[-1])[rows]
    if flat.dtype != torch.uint8:
        return flat.float()
    codes = flat[..., :512].contiguous().view(torch.float8_e4m3fn).float()
    scale = flat[..., 512:528].contiguous().view(torch.float32)
    return codes * scale.repeat_interleave(128, dim=-1)


def _plain_chunk(st):
    new, cached = _ints(st["case"]["new"]), _ints(st["case"]["cached"])
    longest, keys = max(new), max(n + c for n, c in zip(new, cached))
    table, q_start, kv_len = st["page_table"], st["q_start"].long(), st["kv_len"].long()
    # the batch padded to its longest chunk and its longest cache
    pos = torch.arange(keys, device="cuda")
    rows = table.long().clamp_min(0)[:, pos // PAGE] * PAGE + pos % PAGE
    valid = pos[None] < kv_len[:, None]
    lat = torch.where(valid[:, :, None], _row_values(st, rows), 0.0)
    local = torch.arange(longest, device="cuda")
    token = torch.minimum(q_start[:-1, None] + local[None], q_start[1:, None] - 1)
    q = st["q"][token].float().permute(0, 2, 1, 3)
    k = torch.matmul(lat[:, None, :, :LATENT], st["w_uk"].float().transpose(1, 2)[None])
    score = torch.matmul(q[..., :st["dn"]], k.transpose(2, 3))
    del k
    if st["dr"]:
        score += torch.matmul(q[..., st["dn"]:], lat[:, None, :, LATENT:].transpose(2, 3))
    sees = torch.minimum(kv_len[:, None], st["q_pos"].long()[token] + 1)
    score.mul_(st["scale"]).masked_fill_((pos >= sees[:, :, None])[:, None], -math.inf)
    peak = score.amax(dim=3, keepdim=True)
    score.sub_(torch.where(torch.isinf(peak), 0.0, peak)).exp_()
    total = score.sum(dim=3, keepdim=True)
    v = torch.matmul(lat[:, None, :, :LATENT], st["w_uv"].float().transpose(1, 2)[None])
    out = torch.matmul(score, v) / torch.where(total > 0, total, 1.0)
    t = torch.arange(st["q"].shape[0], device="cuda")
    seq = torch.searchsorted(q_start[1:], t, right=True)
    return {"out": out[seq, :, t - q_start[seq]].to(torch.bfloat16)}


def _rms(x):
    return x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS)


def _plain_norm(st):
    b = st["y"].float()
    if st["post"] is not None:
        b = _rms(b) * st["post"].float()
    if st["gate"] is not None:
        b = b * st["gate"].float()
    h = st["residual"].float() + st["scale"] * b
    got = {"residual": h.to(st["residual"].dtype)}
    if st["pre"] is not None:
        got["x"] = (_rms(h) * st["pre"].float()).to(torch.bfloat16)
    return got


def _plain_plan(st):
    cached, new, table, tokens = st["cached_len"].long(), st["new_len"].long(), st["page_table"], st["tokens"]
    kv_len = cached + new
    first, last = (cached + PAGE - 1) // PAGE, (kv_len + PAGE - 1) // PAGE
    taken = torch.cumsum(last - first, 0)
    q_start = torch.nn.functional.pad(torch.cumsum(new, 0), (1, 0))
    column = torch.arange(table.shape[1], device="cuda")
    grown = (column >= first[:, None]) & (column < last[:, None])
    nth = (taken - (last - first))[:, None] + column - first[:, None]
    free = st["free_pages"]
    at = (st["free_count"].long() - 1 - nth).clamp(0, free.numel() - 1)
    table = torch.where(grown, free[at], table)
    t = torch.arange(tokens, device="cuda")
    real = t < q_start[-1]
    seq = torch.searchsorted(q_start[1:], t, right=True).clamp_max(len(cached) - 1)
    pos = cached[seq] + t - q_start[seq]
    slot = table[seq, (pos // PAGE).clamp_max(table.shape[1] - 1)].long() * PAGE + pos % PAGE
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return {"q_start": i32(q_start), "kv_len": i32(kv_len), "seq_id": i32(torch.where(real, seq, -1)),
            "q_pos": i32(torch.where(real, pos, -1)), "slot": i32(torch.where(real, slot, -1)),
            "page_table": i32(table), "free_left": i32(st["free_count"].long() - taken[-1:])}


def run(state):
    op = state["op"]
    if own:
        got = state["launch"]()
        if op == "chunk":
            return {"out": got}
        if op == "norm":
            return {"residual": got[0], "x": got[1]} if state["pre"] is not None else {"residual": got[0]}
        return {"q_start": got.q_start, "kv_len": got.kv_len, "seq_id": got.seq_id, "q_pos": got.q_pos, "slot": got.slot,
                "page_table": got.page_table, "free_left": got.free_left}
    return {"chunk": _plain_chunk, "norm": _plain_norm, "plan": _plain_plan}[op](state)


# ------------------------------------------------------------------------------------- definition in 64 bits


def _exact_chunk(case, seed):
    """The same attention with the weights folded into the query and the output instead: scores of
    the folded query with the latent rows themselves, sums of latent rows, then the value weights."""
    st = _prepare_chunk(case, seed)
    heads, dn, dr = case["heads"], st["dn"], st["dr"]
    out = torch.zeros((st["q"].shape[0], heads, st["dv"]), dtype=torch.float64, device="cuda")
    start = 0
    for s, (n, c) in enumerate(zip(_ints(case["new"]), _ints(case["cached"]))):
        page = st["page_table"][s].tolist()
        flat = st["kv"].view(-1, st["kv"].shape[-1])
        rows = torch.cat([flat[p * PAGE:p * PAGE + PAGE] for p in page if p >= 0])[:n + c]
        if rows.dtype == torch.uint8:
            codes = rows[:, :512].contiguous().view(torch.float8_e4m3fn).double().view(-1, 4, 128)
            rows = (codes * rows[:, 512:528].contiguous().view(torch.float32).double()[:, :, None]).reshape(-1, 512)
        rows = rows.double()
        # one more key for each later token of the chunk
        first = torch.arange(c + 1, n + c + 1, device="cuda")
        step = max(1, 2 ** 27 // (n + c))
        for h in range(heads):
            w_uk, w_uv = st["w_uk"][h].double(), st["w_uv"][h].double()
            for a in range(0, n, step):
                q = st["q"][start + a:start + min(n, a + step), h].double()
                score = (q[:, :dn] @ w_uk) @ rows[:, :LATENT].T
                if dr:
                    score += q[:, dn:] @ rows[:, LATENT:].T
                score *= st["scale"]
                hidden = torch.arange(n + c, device="cuda")[None] >= first[a:a + step, None]
                score[hidden] = -math.inf
                p = torch.softmax(score, dim=1)
                out[start + a:start + min(n, a + step), h] = (p @ rows[:, :LATENT]) @ w_uv.T
        start += n
    return {"out": out}


def _exact_norm(case, seed):
    st = _prepare_norm(case, seed)
    d = case["width"]
    b = st["y"].double()
    if st["post"] is not None:
        b = b / torch.sqrt(b.square().sum(1, keepdim=True) / d + EPS) * st["post"].double()
    if st["gate"] is not None:
        b = st["gate"].double() * b
    h = st["residual"].double() + st["scale"] * b
    got = {"residual": h}
    if st["pre"] is not None:
        got["x"] = h / torch.sqrt(h.square().sum(1, keepdim=True) / d + EPS) * st["pre"].double()
    return got


def exact(case, seed):
    """The step plan's outputs are whole numbers: they are compared as they are."""
    if case["op"] == "chunk":
        return _exact_chunk(case, seed)
    return _exact_norm(case, seed) if case["op"] == "norm" else None


# ------------------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["op"] == "chunk":
        _, dr, dn, dv, row_bytes = FORMATS[case["rows"]]
        payload = 528 if case["rows"] == "fp8" else row_bytes
        heads, flops, nbytes = case["heads"], 0, 2 * case["heads"] * LATENT * (dn + dv)
        for n, c in zip(_ints(case["new"]), _ints(case["cached"])):
            pairs = n * c + n * (n + 1) // 2
            # keys and values expanded once per cached row, or the weights folded into each query
            # token and its output: whichever form does less work
            expanded = (n + c) * 2 * LATENT * (dn + dv) + pairs * 2 * (dn + dr + dv)
            folded = n * 2 * LATENT * (dn + dv) + pairs * 2 * (2 * LATENT + dr)
            flops += heads * min(expanded, folded)
            nbytes += (n + c) * payload + n * heads * 2 * (dn + dr + dv) + 4 * (n + -(-(n + c) // PAGE))
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "norm":
        t, d = case["tokens"], case["width"]
        each = 2 + 2 * (4 if case["residual"] == "f32" else 2) + (2 if case["pre"] else 0) + (2 if case["gate"] == "token" else 0)
        once = 2 * ((1 if case["post"] else 0) + (1 if case["pre"] else 0) + (1 if case["gate"] == "channel" else 0))
        return {"bytes": t * d * each + d * once, "flops": t * d * 10}
    n, tokens = case["requests"], case["requests"] - case["chunks"] + case["chunks"] * case["chunk"]
    grown = (tokens + n) // PAGE  # pages, about
    return {"bytes": 16 * n + 12 * (tokens + case["padding"]) + 8 * grown, "flops": tokens}
