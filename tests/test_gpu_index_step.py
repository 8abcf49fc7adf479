"""GPU: the index branch as a sparse step uses it: write -> scores -> select -> attention, in both forms;
captured and replayed with new contents; on other streams and many at once; batches padded to a captured
size; empty calls.

The selection is checked against the oracle on the scores that the device made (whole numbers), the
scores and the attention against theirs (``test_gpu_index``, ``conftest.assert_parity``)."""

import math

import numpy as np
import pytest
import torch

from conftest import assert_parity
from oracle import fp8 as ofp8
from oracle import index as oindex
from oracle import mla as omla
from test_gpu_index import PAGE, ROW, batch, bf16, check_rows, host, i32
from tq_mla import _abi, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


class Step:
    """A layer's caches of some requests, filled by the writers, and one step over them."""

    def __init__(self, device, seed, new, lens, fmt, heads=64, index_heads=32, tokens=None):
        rng = np.random.default_rng(seed)
        self.dev, self.fmt, self.new, self.lens = device, fmt, list(new), list(lens)
        self.table, self.seq, self.pos, pages = batch(rng, new, lens)
        t = len(self.seq)
        self.tokens = t if tokens is None else tokens
        pad = self.tokens - t
        self.seq = np.concatenate([self.seq, np.full(pad, -1)])
        self.pos = np.concatenate([self.pos, np.full(pad, -1)])
        self.d_table, self.d_kv_len = i32(self.table, device), i32(lens, device)
        self.d_seq, self.d_pos = i32(self.seq, device), i32(self.pos, device)
        width = 576 if fmt == _abi.KV_BF16_ROPE576 else 512
        row = {_abi.KV_FP8_E4M3: 544}.get(fmt, 2 * width)
        self.kv = torch.zeros((pages, PAGE, row), dtype=torch.uint8, device=device)
        self.index = torch.zeros((pages, PAGE, ROW), dtype=torch.uint8, device=device)
        freq, mscale = ops.rope_frequencies(64, 10000.0, factor=4.0, original=4096)
        self.kw = dict(scale=index_heads ** -0.5 * 128 ** -0.5, freq=freq.float().to(device), rope_mscale=mscale,
                       norm_weight=bf16(1 + 0.1 * rng.standard_normal(128), device),
                       norm_bias=bf16(0.1 * rng.standard_normal(128), device))
        # what is cached: every row of every request
        cached_seq = i32(np.repeat(np.arange(len(lens)), lens), device)
        cached_pos = i32(np.concatenate([np.arange(n) for n in lens] + [np.zeros(0)]), device)
        n = sum(lens)
        ops.kv_write(bf16(rng.standard_normal((n, width)), device), self.kv, self.d_table, cached_seq, cached_pos, kv_format=fmt)
        key_kw = {k: v for k, v in self.kw.items() if k != "scale"}
        ops.index_write(None, bf16(rng.standard_normal((n, 128)), device), None, self.d_table, cached_seq, cached_pos,
                        self.index, **key_kw)
        self.q = bf16(rng.standard_normal((self.tokens, heads, width)), device)
        self.iq = bf16(rng.standard_normal((self.tokens, index_heads, 128)) * 2, device)
        self.ik = bf16(rng.standard_normal((self.tokens, 128)), device)
        self.iw = bf16(rng.standard_normal((self.tokens, index_heads)), device)
        self.columns = PAGE * self.table.shape[1]
        self.scale = ops.default_scale(width)
        self.flags = torch.zeros(1, dtype=torch.int32, device=device)

    def select(self, k, pages, stream=None, **keep):
        codes, w = ops.index_write(self.iq, self.ik, self.iw, self.d_table, self.d_seq, self.d_pos, self.index,
                                   flags=self.flags, stream=stream, **self.kw)
        scores = ops.index_scores(codes, w, self.index, self.d_table, self.d_seq, self.d_pos, self.d_kv_len,
                                  flags=self.flags, stream=stream)
        idx, length = ops.index_select(scores, self.d_seq, self.d_pos, self.d_kv_len, k, flags=self.flags, stream=stream,
                                       page_table=self.d_table if pages else None, **keep)
        return codes, w, scores, idx, length

    def check_scores(self, codes, w, scores):
        want, mass = oindex.scores(codes.cpu().numpy(), w.cpu().numpy(), self.index.view(-1, ROW).cpu().numpy(), self.table,
                                   self.seq, self.pos, np.array(self.lens), self.columns, np.full((self.tokens, self.columns), -np.inf))
        got = host(scores)
        seen = np.isfinite(want)
        assert np.array_equal(np.isfinite(got), seen)
        assert (np.abs(got[seen] - want[seen]) <= 260 * U * mass[seen]).all()

    def rows(self):
        flat = self.kv.view(-1, self.kv.shape[-1]).cpu()
        if self.fmt == _abi.KV_FP8_E4M3:
            return ofp8.operand_rows(flat.numpy())
        return flat.contiguous().view(torch.bfloat16).double().numpy()


@pytest.mark.parametrize("fmt", [_abi.KV_BF16, _abi.KV_FP8_E4M3])
@pytest.mark.parametrize("new,lens,k", [([1, 1, 1, 1], [37, 700, 3001, 64], 128), ([2, 4, 1, 3], [700, 300, 1000, 3], 257),
                                        ([1], [5000], 2051)])
def test_sparse_step(cuda_device, fmt, new, lens, k):
    s = Step(cuda_device, sum(lens), new, lens, fmt)
    codes, w, scores, idx, length = s.select(k, False)
    out, lse = ops.mla_decode(s.q, s.kv, s.d_table, s.d_seq, s.d_pos, s.d_kv_len, scale=s.scale, query_counts=new, kv_format=fmt,
                              idx=idx, k_len=length, out_dtype=torch.float32)
    torch.cuda.synchronize()
    assert int(s.flags) == 0
    s.check_scores(codes, w, scores)
    want_idx, want_len = oindex.select(scores.cpu().numpy(), s.seq, s.pos, np.array(lens), k)
    np.testing.assert_array_equal(idx.cpu().numpy(), want_idx)
    np.testing.assert_array_equal(length.cpu().numpy(), want_len)
    ref, ref_lse = omla.sparse_attention(host(s.q), s.rows(), s.table, s.seq, s.pos, np.array(lens), want_idx, want_len, scale=s.scale)
    assert_parity(host(out), host(lse), ref, ref_lse)


@pytest.mark.parametrize("fmt", [_abi.KV_BF16_ROPE576, _abi.KV_BF16, _abi.KV_FP8_E4M3])
@pytest.mark.parametrize("new,lens,k,keep", [([1, 1, 1], [40, 2000, 4097], 8, 1), ([3, 1, 2], [1000, 64, 6000], 5, 0), ([1], [129], 1, 0)])
def test_step_over_selected_pages(cuda_device, fmt, new, lens, k, keep):
    s = Step(cuda_device, sum(lens) + 1, new, lens, fmt)
    codes, w, scores, table, length = s.select(k, True, keep_first=keep, keep_last=keep)
    t = s.tokens
    own = i32(np.arange(t), cuda_device)
    out, lse = ops.mla_decode(s.q, s.kv, table, own, s.d_pos, length, scale=s.scale, query_counts=[1] * t, kv_format=fmt,
                              out_dtype=torch.float32)
    torch.cuda.synchronize()
    assert int(s.flags) == 0
    s.check_scores(codes, w, scores)
    want, want_len = oindex.select(scores.cpu().numpy(), s.seq, s.pos, np.array(lens), k, s.table, keep, keep)
    np.testing.assert_array_equal(table.cpu().numpy(), want)
    np.testing.assert_array_equal(length.cpu().numpy(), want_len)
    # the positions that those pages hold, as a selection of rows
    rows, q = s.rows(), host(s.q)
    ref, ref_lse = np.zeros((t, q.shape[1], 512)), np.full((t, q.shape[1]), -np.inf)
    for i in range(t):
        columns = {int(p): c for c, p in enumerate(s.table[s.seq[i]])}
        at = [p * PAGE + r for p in want[i] if p >= 0 for r in range(PAGE) if columns[int(p)] * PAGE + r <= s.pos[i]]
        assert len(at) == want_len[i]
        ref[i], ref_lse[i] = omla.identity_core(q[i], rows[at], s.scale, 512)
    assert_parity(host(out), host(lse), ref, ref_lse)


def test_step_writes_the_rows_that_it_scores(cuda_device):
    """A token's own key is in the cache when its scores are taken."""
    s = Step(cuda_device, 5, [1, 2], [100, 65], _abi.KV_BF16)
    s.select(8, False)
    torch.cuda.synchronize()
    want = oindex.normalised(host(s.ik), host(s.kw["norm_weight"]), host(s.kw["norm_bias"]), 1e-6)
    want = oindex.turned(want, s.pos, host(s.kw["freq"]), 0, False, s.kw["rope_mscale"])
    at, _ = oindex.slots(s.table, s.seq, s.pos, s.index.shape[0])
    got = s.index.view(-1, ROW).cpu().numpy()[at]
    check_rows(got[:, :128], np.ascontiguousarray(got[:, 128:132]).view(np.float32)[:, 0].astype(np.float64), want)


@pytest.mark.parametrize("pages", [False, True])
def test_padded_step_in_a_graph_with_new_contents(cuda_device, pages):
    """Captured once at a padded size; replayed for other lengths, tables and values."""
    fmt = _abi.KV_BF16_ROPE576 if pages else _abi.KV_BF16
    steps = [Step(cuda_device, 60 + i, new, lens, fmt, tokens=8) for i, (new, lens) in
             enumerate([([1, 1, 1], [900, 1000, 64]), ([2, 1, 3], [1000, 10, 333]), ([1, 4, 1], [5, 1024, 700])])]
    s = steps[0]
    columns, k = max(x.table.shape[1] for x in steps), 6 if pages else 100
    pool = max(x.kv.shape[0] for x in steps)
    fixed = dict(table=torch.full((3, columns), -1, dtype=torch.int32, device=cuda_device),
                 kv=torch.zeros((pool, *s.kv.shape[1:]), dtype=torch.uint8, device=cuda_device),
                 index=torch.zeros((pool, *s.index.shape[1:]), dtype=torch.uint8, device=cuda_device))
    names = ("d_seq", "d_pos", "d_kv_len", "q", "iq", "ik", "iw")
    fixed.update({n: getattr(s, n).clone() for n in names})

    def fill(x):
        for n in names:
            fixed[n].copy_(getattr(x, n))
        fixed["table"].fill_(-1)
        fixed["table"][:, :x.table.shape[1]] = x.d_table
        for n in ("kv", "index"):
            fixed[n].zero_()
            fixed[n][:getattr(x, n).shape[0]] = getattr(x, n)

    t = s.tokens
    codes = torch.empty((t, 32, 128), dtype=torch.uint8, device=cuda_device)
    w = torch.empty((t, 32), device=cuda_device)
    scores = torch.full((t, PAGE * columns), -math.inf, device=cuda_device)
    idx = torch.empty((t, k), dtype=torch.int32, device=cuda_device)
    length = torch.empty(t, dtype=torch.int32, device=cuda_device)
    out, lse = torch.empty((t, 64, 512), device=cuda_device), torch.empty((t, 64), device=cuda_device)
    flags = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    where = (fixed["table"], fixed["d_seq"], fixed["d_pos"])
    write = ops.IndexWrite(fixed["iq"], fixed["ik"], fixed["iw"], *where, fixed["index"], codes, w, **s.kw)
    score = ops.IndexScores(codes, w, fixed["index"], *where, fixed["d_kv_len"], scores)
    select = ops.IndexSelect(scores, fixed["d_seq"], fixed["d_pos"], fixed["d_kv_len"], idx, length,
                             page_table=fixed["table"] if pages else None)
    if pages:
        attend = ops.MlaLaunch(fixed["q"], fixed["kv"], idx, i32(np.arange(t), cuda_device), fixed["d_pos"], length, out, lse,
                               scale=s.scale, query_counts=[1] * t, kv_format=fmt)
    else:
        attend = ops.MlaLaunch(fixed["q"], fixed["kv"], fixed["table"], fixed["d_seq"], fixed["d_pos"], fixed["d_kv_len"], out, lse,
                               scale=s.scale, query_counts=[4, 4, 0], kv_format=fmt, idx=idx, k_len=length)

    def step():
        write(flags)
        score(flags)
        select(flags)
        attend()

    fill(s)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for x in steps + steps[:1]:
        fill(x)
        flags.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert int(flags) == _abi.DEV_SEQ_RANGE       # the padded tokens
        got_table = fixed["table"].cpu().numpy()
        want, want_len = oindex.select(scores.cpu().numpy(), x.seq, x.pos, np.array(x.lens), k, got_table if pages else None)
        np.testing.assert_array_equal(idx.cpu().numpy(), want)
        np.testing.assert_array_equal(length.cpu().numpy(), want_len)
        real = x.seq >= 0
        assert (out[torch.from_numpy(~real)] == 0).all() and torch.isneginf(lse[torch.from_numpy(~real)]).all()
        n = int(real.sum())
        rows, q = x.rows(), host(x.q)
        for i in range(n):
            if pages:
                columns_of = {int(p): c for c, p in enumerate(x.table[x.seq[i]])}
                at = [p * PAGE + r for p in want[i] if p >= 0 for r in range(PAGE) if columns_of[int(p)] * PAGE + r <= x.pos[i]]
            else:
                at = [int(x.table[x.seq[i], p // PAGE]) * PAGE + p % PAGE for p in want[i] if p >= 0]
            ref, ref_lse = omla.identity_core(q[i], rows[at], x.scale, 512)
            assert_parity(host(out[i:i + 1]), host(lse[i:i + 1]), ref[None], ref_lse[None])
    del graph


def test_calls_on_a_side_stream(cuda_device):
    """What a one-shot call returns belongs to the stream that it was given, and is what it gives otherwise."""
    from test_gpu_side_streams import owner
    s = Step(cuda_device, 7, [1, 3, 1], [700, 2000, 90], _abi.KV_BF16)
    want = s.select(100, False) + s.select(5, True)[3:]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = s.select(100, False, stream=side) + s.select(5, True, stream=side)[3:]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert owner(a) == side.cuda_stream
        assert torch.equal(a, b)


def test_calls_on_many_streams_at_once(cuda_device):
    """Calls of all forms beside each other and beside the attention, launched and replayed: each gives the
    bits that it gives alone."""
    steps = [Step(cuda_device, 80, [1] * 40, [900 + 50 * i for i in range(40)], _abi.KV_BF16, heads=16),
             Step(cuda_device, 81, [300], [3000], _abi.KV_BF16, heads=16, index_heads=48),
             Step(cuda_device, 82, [1, 2], [30000, 20000], _abi.KV_BF16_ROPE576, heads=16, index_heads=8),
             Step(cuda_device, 83, [700, 33], [2500, 100], _abi.KV_FP8_E4M3, heads=16, index_heads=128)]
    ks = [(64, False), (512, False), (40, True), (300, False)]
    calls, outputs = [], []
    for s, (k, pages) in zip(steps, ks):
        t, h = s.iq.shape[:2]
        codes, w, scores, idx, length = (x.clone() for x in s.select(k, pages))
        launch = [ops.IndexWrite(s.iq, s.ik, s.iw, s.d_table, s.d_seq, s.d_pos, s.index, codes, w, **s.kw),
                  ops.IndexScores(codes, w, s.index, s.d_table, s.d_seq, s.d_pos, s.d_kv_len, scores),
                  ops.IndexSelect(scores, s.d_seq, s.d_pos, s.d_kv_len, idx, length, page_table=s.d_table if pages else None)]
        own = i32(np.arange(t), cuda_device)
        if pages:
            out, lse = torch.empty((t, 16, 512), device=cuda_device), torch.empty((t, 16), device=cuda_device)
            launch.append(ops.MlaLaunch(s.q, s.kv, idx, own, s.d_pos, length, out, lse, scale=s.scale, query_counts=[1] * t,
                                        kv_format=s.fmt))
        calls.append(launch)
        outputs.append((codes, w, scores, idx, length))
    torch.cuda.synchronize()
    want = [[x.clone() for x in o] for o in outputs]
    streams, graphs = [torch.cuda.Stream() for _ in calls], []
    for launch, stream in zip(calls, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            for call in launch:
                call()
        graphs.append(graph)
    rng = np.random.default_rng(9)
    torch.cuda.synchronize()
    for k in range(300):
        if k % 30 == 0:
            for codes, w, scores, idx, length in outputs:
                codes.zero_(), w.zero_(), idx.fill_(7), length.zero_()
            torch.cuda.synchronize()
        for _ in range(4):
            for i in rng.permutation(len(calls)):
                with torch.cuda.stream(streams[i]):
                    if rng.random() < 0.5:
                        graphs[i].replay()
                    else:
                        for call in calls[i]:
                            call()
        torch.cuda.synchronize()
        if k % 10 == 9:
            for got, ref in zip(outputs, want):
                assert all(torch.equal(a, b) for a, b in zip(got, ref))
    del graph
    graphs.clear()


def test_calls_without_tokens(cuda_device):
    e = torch.empty(0, dtype=torch.int32, device=cuda_device)
    table, kv_len = i32([[0, 1]], cuda_device), i32([100], cuda_device)
    index = torch.full((2, PAGE, ROW), 3, dtype=torch.uint8, device=cuda_device)
    q = torch.empty((0, 16, 128), dtype=torch.bfloat16, device=cuda_device)
    w_in = torch.empty((0, 16), dtype=torch.bfloat16, device=cuda_device)
    codes, w = ops.index_write(q, q[:, 0], w_in, table, e, e, index)
    scores = ops.index_scores(codes, w, index, table, e, e, kv_len)
    idx, length = ops.index_select(scores, e, e, kv_len, 5)
    torch.cuda.synchronize()
    assert codes.shape == (0, 16, 128) and scores.shape == (0, 128) and idx.shape == (0, 5) and length.shape == (0,)
    assert (index == 3).all()


def test_a_pool_without_pages(cuda_device):
    """Every page is outside it: rows read as zeros."""
    index = torch.empty((0, PAGE, ROW), dtype=torch.uint8, device=cuda_device)
    codes = torch.full((2, 16, 128), 0x38, dtype=torch.uint8, device=cuda_device)
    w, flags = torch.ones((2, 16), device=cuda_device), torch.zeros(1, dtype=torch.int32, device=cuda_device)
    scores = ops.index_scores(codes, w, index, i32([[0, 0]], cuda_device), i32([0, 0], cuda_device), i32([70, 99], cuda_device),
                              i32([100], cuda_device), flags=flags)
    torch.cuda.synchronize()
    assert int(flags) == _abi.DEV_PAGE_RANGE
    assert (scores[0, :71] == 0).all() and (scores[1, :100] == 0).all() and torch.isneginf(scores[1, 100:]).all()


def test_flags_that_are_not_int32_on_the_device_are_refused(cuda_device):
    s = Step(cuda_device, 11, [1], [70], _abi.KV_BF16)
    for flags in (torch.zeros(1, device=cuda_device), torch.zeros(1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32, device=cuda_device)):
        with pytest.raises(ValueError):
            ops.index_write(s.iq, s.ik, s.iw, s.d_table, s.d_seq, s.d_pos, s.index, flags=flags, **s.kw)
        with pytest.raises(ValueError):
            ops.index_select(torch.zeros((1, 70), device=cuda_device), s.d_seq, s.d_pos, s.d_kv_len, 3, flags=flags)
