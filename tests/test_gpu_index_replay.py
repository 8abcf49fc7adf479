"""GPU: a captured step of the index branch whose outputs are reset before each replay: every stage is
compared with its oracle, so that a stage that did nothing or read what an earlier replay left is seen; and
the same for calls of several steps beside each other. Tolerances: see ``test_gpu_index``."""

import numpy as np
import pytest
import torch

from conftest import assert_parity
from oracle import index as oindex
from oracle import mla as omla
from test_gpu_index import PAGE, ROW, U, check_rows, host, i32
from test_gpu_index_step import Step
from tq_mla import _abi, ops

pytestmark = pytest.mark.gpu


class Calls:
    """The four calls of a step on buffers of their own."""

    def __init__(self, device, s, k, pages, columns=None, pool=None, sequences=None, counts=None):
        self.k, self.pages, self.kw, self.fmt, self.scale = k, pages, s.kw, s.fmt, s.scale
        self.flags = torch.zeros(1, dtype=torch.int32, device=device)
        columns = s.table.shape[1] if columns is None else columns
        pool = s.kv.shape[0] if pool is None else pool
        t, heads, index_heads = s.tokens, s.q.shape[1], s.iq.shape[1]
        ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)  # noqa: E731
        self.table, self.seq, self.pos, self.kv_len = ints(len(s.lens), columns), ints(t), ints(t), ints(len(s.lens))
        self.kv = torch.zeros((pool, *s.kv.shape[1:]), dtype=torch.uint8, device=device)
        self.index = torch.zeros((pool, PAGE, ROW), dtype=torch.uint8, device=device)
        self.q, self.iq, self.ik, self.iw = (torch.zeros_like(x) for x in (s.q, s.iq, s.ik, s.iw))
        self.codes = torch.empty((t, index_heads, 128), dtype=torch.uint8, device=device)
        self.w = torch.empty((t, index_heads), device=device)
        self.scores = torch.empty((t, PAGE * columns), device=device)
        self.idx, self.length = ints(t, k), ints(t)
        self.out, self.lse = torch.empty((t, heads, 512), device=device), torch.empty((t, heads), device=device)
        where = (self.table, self.seq, self.pos)
        counts = s.new if counts is None else counts
        self.calls = [ops.IndexWrite(self.iq, self.ik, self.iw, *where, self.index, self.codes, self.w, **s.kw),
                      ops.IndexScores(self.codes, self.w, self.index, *where, self.kv_len, self.scores),
                      ops.IndexSelect(self.scores, self.seq, self.pos, self.kv_len, self.idx, self.length,
                                      page_table=self.table if pages else None)]
        if pages:
            self.attend = ops.MlaLaunch(self.q, self.kv, self.idx, i32(np.arange(t), device), self.pos, self.length, self.out, self.lse,
                                        scale=s.scale, query_counts=[1] * t, kv_format=s.fmt)
        else:
            self.attend = ops.MlaLaunch(self.q, self.kv, *where, self.kv_len, self.out, self.lse, scale=s.scale, query_counts=counts,
                                        kv_format=s.fmt, idx=self.idx, k_len=self.length)

    def fill(self, s):
        """The inputs of step ``s``, and outputs that no stage would leave."""
        self.table.fill_(-1)
        self.table[:, :s.table.shape[1]] = s.d_table
        for mine, its in ((self.seq, s.d_seq), (self.pos, s.d_pos), (self.kv_len, s.d_kv_len), (self.q, s.q), (self.iq, s.iq),
                          (self.ik, s.ik), (self.iw, s.iw)):
            mine.copy_(its)
        self.kv.zero_()
        self.kv[:s.kv.shape[0]] = s.kv
        self.index.zero_()
        self.index[:s.index.shape[0]] = s.index
        rows, _ = oindex.slots(s.table, s.seq, s.pos, s.index.shape[0])
        self.index.view(-1, ROW)[torch.from_numpy(rows[rows >= 0])] = 0x7F           # NaN, until they are written
        self.reset()

    def reset(self):
        self.flags.zero_()
        self.codes.fill_(0x7F)
        self.w.fill_(np.nan)
        self.scores.fill_(-np.inf)
        self.idx.fill_(7)
        self.length.fill_(-9)
        self.out.fill_(np.nan)
        self.lse.fill_(np.nan)

    def __call__(self):
        for call in self.calls:
            call(self.flags)
        self.attend()

    def check(self, s):
        """Every stage against its oracle on what the stage before gave."""
        real = s.seq >= 0
        assert int(self.flags) == (0 if real.all() else _abi.DEV_SEQ_RANGE)
        freq, mscale = host(self.kw["freq"]), self.kw["rope_mscale"]
        want_q = oindex.turned(host(s.iq), s.pos, freq, 0, False, mscale)
        scale = np.abs(want_q).max(axis=-1) / 448.0
        check_rows(self.codes.cpu().numpy(), scale, want_q)
        np.testing.assert_allclose(host(self.w), host(s.iw) * np.float32(self.kw["scale"]) * scale, rtol=64 * U + 3 * U)
        keys = oindex.normalised(host(s.ik), host(self.kw["norm_weight"]), host(self.kw["norm_bias"]), 1e-6)
        keys = oindex.turned(keys, s.pos, freq, 0, False, mscale)[real]
        rows, _ = oindex.slots(s.table, s.seq, s.pos, s.index.shape[0])
        flat = self.index.view(-1, ROW).cpu().numpy()
        got = flat[rows[real]]
        check_rows(got[:, :128], np.ascontiguousarray(got[:, 128:132]).view(np.float32)[:, 0].astype(np.float64), keys)
        want, mass = oindex.scores(self.codes.cpu().numpy(), host(self.w), flat, s.table, s.seq, s.pos, np.array(s.lens),
                                   self.scores.shape[1], np.full(self.scores.shape, -np.inf))
        seen = np.isfinite(want)
        scores = host(self.scores)
        assert np.array_equal(np.isfinite(scores), seen) and np.isneginf(scores[~seen]).all()
        assert (np.abs(scores[seen] - want[seen]) <= 260 * U * mass[seen]).all()
        picked, count = oindex.select(self.scores.cpu().numpy(), s.seq, s.pos, np.array(s.lens), self.k,
                                      self.table.cpu().numpy() if self.pages else None)
        np.testing.assert_array_equal(self.idx.cpu().numpy(), picked)
        np.testing.assert_array_equal(self.length.cpu().numpy(), count)
        pool, q = s.rows(), host(s.q)
        ref, ref_lse = np.zeros(self.out.shape), np.full(self.lse.shape, -np.inf)
        for i in np.flatnonzero(real):
            if self.pages:
                columns_of = {int(p): c for c, p in enumerate(s.table[s.seq[i]])}
                at = [p * PAGE + r for p in picked[i] if p >= 0 for r in range(PAGE) if columns_of[int(p)] * PAGE + r <= s.pos[i]]
            else:
                at = [int(s.table[s.seq[i], p // PAGE]) * PAGE + p % PAGE for p in picked[i] if p >= 0]
            ref[i], ref_lse[i] = omla.identity_core(q[i], pool[at], s.scale, 512)
        assert_parity(host(self.out), host(self.lse), ref, ref_lse)

    def outputs(self):
        return self.codes, self.w, self.index, self.scores, self.idx, self.length, self.out, self.lse


@pytest.mark.parametrize("pages", [False, True])
def test_every_stage_of_a_replayed_step(cuda_device, pages):
    fmt = _abi.KV_BF16_ROPE576 if pages else _abi.KV_BF16
    steps = [Step(cuda_device, 160 + i, new, lens, fmt, tokens=8) for i, (new, lens) in
             enumerate([([1, 1, 1], [900, 1000, 64]), ([2, 1, 3], [1000, 10, 333]), ([1, 4, 1], [5, 1024, 700])])]
    calls = Calls(cuda_device, steps[0], 6 if pages else 100, pages, columns=max(s.table.shape[1] for s in steps),
                  pool=max(s.kv.shape[0] for s in steps), counts=[4, 4, 0])
    for s in steps:          # (the norm and the frequencies are the captured call's)
        s.kw = calls.kw
    calls.fill(steps[0])
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for s in steps + steps[:1]:
        calls.fill(s)
        graph.replay()
        torch.cuda.synchronize()
        calls.check(s)
    del graph


def test_every_stage_of_steps_beside_each_other(cuda_device):
    """Steps of different forms on streams of their own, launched or replayed in turn: each stage is the
    oracle's alone, and gives the same bits beside the others."""
    forms = [(Step(cuda_device, 180, [1] * 12, [900 + 50 * i for i in range(12)], _abi.KV_BF16, heads=16), 64, False),
             (Step(cuda_device, 181, [3, 2], [700, 900], _abi.KV_FP8_E4M3, heads=16, index_heads=48), 300, False),
             (Step(cuda_device, 182, [1, 2], [9000, 5000], _abi.KV_BF16_ROPE576, heads=16, index_heads=8), 20, True),
             (Step(cuda_device, 183, [4, 1, 1], [500, 100, 1], _abi.KV_BF16, heads=16, index_heads=128), 5, True)]
    all_calls, want, streams, graphs = [], [], [], []
    for s, k, pages in forms:
        calls = Calls(cuda_device, s, k, pages)
        calls.fill(s)
        calls()
        torch.cuda.synchronize()
        calls.check(s)
        all_calls.append(calls)
        want.append([x.clone() for x in calls.outputs()])
        streams.append(torch.cuda.Stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[-1]):
            calls()
        graphs.append(graph)
    rng = np.random.default_rng(9)
    for _ in range(30):
        for (s, _, _), calls in zip(forms, all_calls):
            calls.fill(s)
        torch.cuda.synchronize()
        for _ in range(3):
            for i in rng.permutation(len(all_calls)):
                with torch.cuda.stream(streams[i]):
                    if rng.random() < 0.5:
                        graphs[i].replay()
                    else:
                        all_calls[i]()
        torch.cuda.synchronize()
        for calls, ref in zip(all_calls, want):
            assert int(calls.flags) == 0
            assert all(torch.equal(a, b) for a, b in zip(calls.outputs(), ref))
    del graph
    graphs.clear()
