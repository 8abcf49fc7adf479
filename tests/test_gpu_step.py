"""GPU: the step plan and the block norm against their oracles.

The plan's outputs are whole numbers and have to be equal. The norm's tolerances: an output is
rounded once, by at most half a step of its type (2^-8 of the value for bf16, 2^-24 for f32), and
what enters it carries f32 roundings (u = 2^-24 each): a sum of squares adds at most 32 values a
thread and then a tree and a row of at most 37 terms, halved by the square root, and a handful of
products follow, so a norm's factor is off by less than 64 u of itself."""

import numpy as np
import pytest
import torch

from oracle import step as ostep
from tq_mla import _abi, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
FACTOR = 64 * U


def _i32(a, device):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(device)


def _step(rng, requests, cached, new, columns, spare=5):
    """A batch whose requests hold the pages of their cached tokens; all others are free."""
    held = -(-np.maximum(cached, 0) // 64)
    order = rng.permutation(requests * columns + spare)
    table = np.full((requests, columns), -7)
    for s in range(requests):
        n = min(held[s], columns)
        table[s, :n] = order[s * columns:s * columns + n]
    used = set(table[table >= 0].tolist())
    return table, np.array([p for p in order if p not in used])


def _check_plan(device, cached, new, table, free, count, tokens, launch=None):
    flags = torch.zeros(1, dtype=torch.int32, device=device)
    d_table = _i32(table, device)
    args = (_i32(cached, device), _i32(new, device), d_table, _i32(free, device), _i32([count], device))
    got = ops.step_plan(*args, tokens=tokens, flags=flags)
    torch.cuda.synchronize()
    want = ostep.step_plan(cached, new, table, free, count, tokens)
    for name, ref in zip(("q_start", "kv_len", "seq_id", "q_pos", "slot", "page_table"), want):
        np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), ref, err_msg=name)
    assert int(got.free_left) == want[6] and int(flags) == want[7]


@pytest.mark.parametrize("requests,longest,cached_to,padding", [
    (1, 1, 1, 0), (1, 200, 64, 3), (3, 2, 130, 1), (64, 1, 8192, 0), (33, 300, 700, 17),
    (1024, 3, 90, 5), (1025, 7, 256, 0), (4096, 4, 200, 100), (9001, 2, 65, 9), (40, 3000, 5000, 77)])
def test_plan_of_random_lengths(cuda_device, requests, longest, cached_to, padding):
    rng = np.random.default_rng(requests)
    cached = rng.integers(0, cached_to + 1, requests)
    new = rng.integers(0, longest + 1, requests)
    columns = (cached_to + longest + 63) // 64 + 1
    table, free = _step(rng, requests, cached, new, columns)
    _check_plan(cuda_device, cached, new, table, free, len(free), int(new.sum()) + padding)


@pytest.mark.parametrize("case", ["borders", "nothing new", "all empty", "negative", "short table",
                                  "cached past the table", "empty pool", "pool of two", "too many tokens",
                                  "count past the pool", "negative count", "no token rows"])
def test_plan_at_its_edges(cuda_device, case):
    rng = np.random.default_rng(5)
    cached = np.array([0, 63, 64, 65, 128, 1, 127])
    new = np.array([64, 1, 1, 63, 0, 127, 2])
    columns, tokens = 4, 300
    if case == "nothing new":
        new = np.zeros_like(new)
    if case == "all empty":
        cached, new = np.zeros_like(new), np.zeros_like(new)
    if case == "negative":
        cached, new = np.array([0, -3, 64, 65, 128, 1, 127]), np.array([64, 2, -1, 63, 0, 127, 2])
    if case == "short table":
        new = np.array([64, 1, 400, 63, 0, 127, 200])
        tokens = 900
    if case == "cached past the table":
        cached = np.array([0, 63, 64, 300, 128, 1, 127])
    table, free = _step(rng, len(new), cached, new, columns)
    count = len(free)
    if case == "empty pool":
        count = 0
    if case == "pool of two":
        count = 2
    if case == "too many tokens":
        tokens = 100
    if case == "count past the pool":
        count += 11
    if case == "negative count":
        count = -4
    if case == "no token rows":
        tokens = 0
    _check_plan(cuda_device, cached, new, table, free, count, tokens)


@pytest.mark.parametrize("requests,tokens", [(300, 1 << 19), (5000, 70000)])
def test_plan_past_the_near_kernel(cuda_device, requests, tokens):
    """Many requests, or many token rows: the scan that is split over clusters."""
    rng = np.random.default_rng(requests)
    cached, new = rng.integers(0, 300, requests), rng.integers(0, 20, requests)
    table, free = _step(rng, requests, cached, new, 6)
    _check_plan(cuda_device, cached, new, table, free, len(free) - 40, tokens)


def test_plan_of_lengths_near_the_type_border(cuda_device):
    top = 2 ** 31 - 1
    cached, new = np.array([top, 5, top - 1]), np.array([3, top, 2])
    table = np.arange(9).reshape(3, 3)
    _check_plan(cuda_device, cached, np.array([3, 4, 2]), table, np.arange(20, 30), 10, 12)
    got = ops.step_plan(_i32(cached, cuda_device), _i32(new, cuda_device), _i32(table, cuda_device),
                        _i32([40], cuda_device), _i32([1], cuda_device), tokens=10)
    assert got.q_start.tolist() == [0, 3, 10, 10] and got.kv_len.tolist() == [192, 128, 192]
    assert got.q_pos.tolist() == [top] * 3 + list(range(5, 12))   # positions past 31 bits stay at the top


def test_plan_of_no_requests(cuda_device):
    e = torch.empty(0, dtype=torch.int32, device=cuda_device)
    got = ops.step_plan(e, e, e.view(0, 3), _i32([4, 5], cuda_device), _i32([2], cuda_device), tokens=3)
    assert got.q_start.tolist() == [0] and got.seq_id.tolist() == [-1] * 3 and int(got.free_left) == 2


def test_plan_replays_from_a_graph_and_chains(cuda_device):
    """A captured plan replayed with other lengths, each step starting from the last one's results."""
    rng = np.random.default_rng(9)
    requests, columns, tokens = 50, 12, 700
    cached, new = np.zeros(requests, np.int64), rng.integers(1, 9, requests)
    table, free = _step(rng, requests, cached, new, columns)
    count = len(free)
    d = [_i32(a, cuda_device) for a in (cached, new, table, free, [count])]
    plan = ops.StepPlan(*d, tokens=tokens)
    plan()                                       # loads the kernel before the capture
    torch.cuda.synchronize()
    d[2].copy_(_i32(table, cuda_device))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan()
    for step in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = ostep.step_plan(cached, new, table, free, count, tokens)
        for name, ref in zip(("q_start", "kv_len", "seq_id", "q_pos", "slot", "page_table"), want):
            np.testing.assert_array_equal(getattr(plan.tables, name).cpu().numpy(), ref, err_msg=name)
        cached, table, count = want[1], want[5], want[6]
        assert int(plan.tables.free_left) == count
        new = rng.integers(0, 2 + 4 * step, requests)
        d[0].copy_(plan.tables.kv_len)
        d[1].copy_(_i32(new, cuda_device))
        d[4].copy_(plan.tables.free_left)
    del graph


def _bf16(a, device):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(torch.bfloat16).to(device)


def _host(t):
    return None if t is None else t.double().cpu().numpy()


def _norm_inputs(seed, rows, width, kind, gate, post, pre, device):
    rng = np.random.default_rng(seed)
    t = {"y": _bf16(rng.standard_normal((rows, width)), device),
         "residual": _bf16(3 * rng.standard_normal((rows, width)), device).to(kind) if kind == torch.bfloat16
         else torch.from_numpy((3 * rng.standard_normal((rows, width))).astype(np.float32)).to(device),
         "gate": {None: None, "channel": _bf16(rng.uniform(-1, 1, width), device),
                  "token": _bf16(rng.uniform(-1, 1, (rows, width)), device)}[gate],
         "post_weight": _bf16(rng.uniform(0.5, 1.5, width), device) if post else None,
         "pre_weight": _bf16(rng.uniform(0.5, 1.5, width), device) if pre else None}
    return t


def _check_norm(t, out, x, scale, eps=1e-6):
    h = {k: _host(v) for k, v in t.items()}
    ref, ref_x = ostep.block_norm(h["y"], h["residual"], post_weight=h["post_weight"], gate=h["gate"],
                                  scale=scale, pre_weight=h["pre_weight"], eps=eps)
    half = 2.0 ** -8 if out.dtype == torch.bfloat16 else U
    carried = (FACTOR + 8 * U) * np.abs(ref - h["residual"]) + 2 * U * np.abs(ref)
    err = np.abs(_host(out) - ref)
    assert (err <= half * np.abs(ref) * (1 + 2.0 ** -8) + carried).all(), float((err - carried).max())
    if ref_x is None:
        assert x is None
        return
    r = 1 / np.sqrt((ref * ref).mean(axis=1, keepdims=True) + eps)
    # an element's own carried error, and the factor's: half the relative error of the mean square
    mean_off = (carried * np.abs(ref)).mean(axis=1, keepdims=True) * r * r
    carried_x = carried * r * np.abs(h["pre_weight"]) + np.abs(ref_x) * (FACTOR + 8 * U + mean_off)
    err = np.abs(_host(x) - ref_x)
    assert (err <= 2.0 ** -8 * np.abs(ref_x) * (1 + 2.0 ** -8) + carried_x * (1 + 2.0 ** -7)).all()


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,width", [(1, 8), (1, 7168), (3, 1024), (64, 4096), (37, 5192), (5, 32768),
                                        (2, 16392), (257, 520)])
@pytest.mark.parametrize("gate,post,pre", [(None, False, True), ("channel", True, True),
                                           ("token", True, False), ("token", False, True)])
def test_norm_against_the_oracle(cuda_device, kind, rows, width, gate, post, pre):
    t = _norm_inputs(rows * width, rows, width, kind, gate, post, pre, cuda_device)
    out, x = ops.block_norm(**t, scale=0.7)
    _check_norm(t, out, x, 0.7)


def test_norm_in_place_and_with_padded_rows(cuda_device):
    rows, width = 19, 1160
    t = _norm_inputs(1, rows, width, torch.bfloat16, "token", True, True, cuda_device)
    ref_in = {k: v.clone() for k, v in t.items()}
    wide = {k: torch.full((rows + 2, width + 24), 9.0, dtype=torch.bfloat16, device=cuda_device)
            for k in ("y", "residual", "gate")}
    for k, w in wide.items():
        w[:rows, :width] = t[k]
        t[k] = w[:rows, :width]
    ops.block_norm(**t, scale=-1.25, out=t["residual"], x=t["y"])     # both written in place
    _check_norm(ref_in, t["residual"], t["y"], -1.25)
    for w in wide.values():                                           # nothing else was written
        assert (w[rows:] == 9.0).all() and (w[:, width:] == 9.0).all()


def test_norm_keeps_what_is_not_finite_in_its_row(cuda_device):
    t = _norm_inputs(2, 6, 640, torch.float32, None, True, True, cuda_device)
    t["y"][1, 5] = float("nan")
    t["residual"][3, 7] = float("inf")
    t["y"][4] = 0
    t["residual"][4] = 0
    out, x = ops.block_norm(**t, scale=1.0)
    assert torch.isnan(out[1]).all() and torch.isnan(x[1]).all()
    assert torch.isinf(out[3, 7]) and torch.isnan(x[3, 7]) and (x[3, :7] == 0).all()
    assert (out[4] == 0).all() and (x[4] == 0).all()
    rows = [0, 2, 5]
    _check_norm({k: (v[rows] if v is not None and v.dim() == 2 else v) for k, v in t.items()}, out[rows], x[rows], 1.0)


def test_norm_of_no_rows_and_on_another_stream(cuda_device):
    e = torch.empty((0, 64), dtype=torch.bfloat16, device=cuda_device)
    w = torch.ones(64, dtype=torch.bfloat16, device=cuda_device)
    out, x = ops.block_norm(e, e.clone(), pre_weight=w)
    assert out.shape == x.shape == (0, 64)
    t = _norm_inputs(3, 300, 2048, torch.bfloat16, "channel", True, True, cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out, x = torch.empty_like(t["residual"]), torch.empty_like(t["y"])
    ops.block_norm(**t, out=out, x=x, scale=0.5, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    _check_norm(t, out, x, 0.5)


def test_refusals_raise(cuda_device):
    t = _norm_inputs(4, 4, 64, torch.bfloat16, None, True, True, cuda_device)
    with pytest.raises(ops.ContractError) as e:
        ops.block_norm(t["y"][:, :60], t["residual"][:, :60])
    assert (e.value.field, e.value.kind) == ("y", 1)
    with pytest.raises(ValueError, match="one CUDA device"):
        ops.block_norm(t["y"], t["residual"].cpu())
    count = _i32([2], cuda_device)
    i = _i32([1, 2], cuda_device)
    with pytest.raises(ops.ContractError) as e:
        ops.step_plan(i, i[:1], _i32(np.zeros((2, 2)), cuda_device), i, count, tokens=3)
    assert (e.value.field, e.value.kind) == ("new_len", 1)
    assert _abi.DEV_POOL_EMPTY == 32
