"""GPU: one-shot calls that are given a stream. What a call allocates belongs to that stream, so that
nothing it still uses is handed to other streams' work when the call returns and drops it; its results
are not handed out again while the caller's stream still reads them."""

import numpy as np
import pytest
import torch

import gpu_helpers as gh
from tq_mla import dist as tdist
from tq_mla import inputs, ops

pytestmark = pytest.mark.gpu


def owner(t):
    """The stream (its handle) that the allocator keeps this tensor's memory for."""
    at = t.data_ptr()
    for segment in torch.cuda.memory_snapshot():
        if segment["address"] <= at < segment["address"] + segment["total_size"]:
            return segment["stream"]
    raise AssertionError("not the caching allocator's memory")


def batch(device, prefill):
    per_seq = 96 if prefill else 1
    w = gh.workload(51, 128, [2500, 900, 3100], per_seq=per_seq)
    b = inputs.materialize(w, device)
    return w, b, (b.q, b.kv, b.page_table, b.seq_id, b.q_pos, b.kv_len)


@pytest.mark.parametrize("prefill", [False, True])
def test_attention_allocates_on_its_stream(cuda_device, prefill, monkeypatch):
    w, b, args = batch(cuda_device, prefill)
    spaces = []

    class Seen(ops.MlaLaunch):
        def __init__(self, *a, **kw):
            super().__init__(*a, **kw)
            spaces.append(owner(self.workspace))

    monkeypatch.setattr(ops, "MlaLaunch", Seen)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    out, lse = ops.mla_decode(*args, scale=w.scale, query_counts=b.query_counts, prefill=prefill, stream=side)
    torch.cuda.synchronize()
    assert [owner(out), owner(lse)] + spaces == [side.cuda_stream] * 3


def test_merges_allocate_on_their_stream(cuda_device):
    side = torch.cuda.Stream()
    parts, lses = torch.randn(3, 5, 16, 512, device=cuda_device), torch.randn(3, 5, 16, device=cuda_device)
    torch.cuda.synchronize()
    out, lse = ops.combine_parts(parts, lses, stream=side)
    torch.cuda.synchronize()
    assert owner(out) == owner(lse) == side.cuda_stream
    want, want_lse = ops.combine_parts(parts, lses)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    comm = tdist.Comm(tdist.Comm.new_id(), 1, 0)
    try:
        wide = torch.randn(5, 16, 1024, device=cuda_device)          # a partial that has to be packed first
        torch.cuda.synchronize()
        out, lse = tdist.context_merge(comm, wide[..., ::2], lses[0], stream=side)
        torch.cuda.synchronize()
        assert owner(out) == owner(lse) == side.cuda_stream
        assert torch.equal(out, wide[..., ::2].to(torch.bfloat16))
    finally:
        comm.destroy()


@pytest.mark.parametrize("prefill", [False, True])
def test_attention_on_another_stream_keeps_its_memory(cuda_device, prefill):
    w, b, args = batch(cuda_device, prefill)
    out = torch.empty((w.tokens, w.heads, 512), dtype=torch.bfloat16, device=cuda_device)
    lse = torch.empty((w.tokens, w.heads), device=cuda_device)
    launch = ops.MlaLaunch(*args, out, lse, scale=w.scale, query_counts=b.query_counts, prefill=prefill)
    launch()
    torch.cuda.synchronize()
    need, want, want_lse = launch.workspace.numel(), out.clone(), lse.clone()
    del launch, out, lse
    side = torch.cuda.Stream()
    for _ in range(3):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        torch.zeros(need, dtype=torch.uint8, device=cuda_device)     # a free block of the current stream
        side.wait_stream(torch.cuda.current_stream())
        outs = []
        for _ in range(4):
            outs.append(ops.mla_decode(*args, scale=w.scale, query_counts=b.query_counts, prefill=prefill,
                                       stream=side))
            torch.full((need,), 255, dtype=torch.uint8, device=cuda_device)
        torch.cuda.synchronize()
        for got, got_lse in outs:
            assert torch.equal(got, want) and torch.equal(got_lse, want_lse)


@pytest.mark.parametrize("call", ["decode", "combine", "norm", "plan"])
def test_results_are_not_reused_while_the_callers_stream_reads_them(cuda_device, call):
    """The caller's stream still has to read a result when the caller drops it, and the call's stream
    then allocates and fills as much memory."""
    w, b, args = batch(cuda_device, False)
    parts, lses = torch.randn(3, 50, 16, 512, device=cuda_device), torch.randn(3, 50, 16, device=cuda_device)
    y = torch.randn(300, 1024, device=cuda_device).to(torch.bfloat16)
    residual = torch.randn(300, 1024, device=cuda_device)
    weight = torch.ones(1024, dtype=torch.bfloat16, device=cuda_device)
    lengths = torch.full((40,), 300, dtype=torch.int32, device=cuda_device)
    table = torch.zeros((40, 30), dtype=torch.int32, device=cuda_device)
    free = torch.arange(4000, dtype=torch.int32, device=cuda_device)
    count = torch.tensor([4000], dtype=torch.int32, device=cuda_device)
    side = torch.cuda.Stream()

    def make():
        if call == "decode":
            return ops.mla_decode(*args, scale=w.scale, query_counts=b.query_counts, stream=side)
        if call == "combine":
            return ops.combine_parts(parts, lses, stream=side)
        if call == "norm":
            return ops.block_norm(y, residual, pre_weight=weight, stream=side)
        got = ops.step_plan(lengths, lengths, table, free, count, tokens=13000, stream=side)
        return got.seq_id, got.q_pos

    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    got = make()
    torch.cuda.synchronize()
    want = [t.clone() for t in got]
    del got
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    got = make()
    here = torch.cuda.current_stream()
    here.wait_stream(side)
    torch.cuda._sleep(200_000_000)              # a tenth of a second of the caller's own work
    copies = [t.clone() for t in got]
    shapes = [(t.shape, t.dtype) for t in got]
    del got
    with torch.cuda.stream(side):
        filled = [torch.full(shape, 99, dtype=dtype, device=cuda_device) for shape, dtype in shapes for _ in range(4)]
    torch.cuda.synchronize()
    for a, z in zip(copies, want):
        assert torch.equal(a, z)
    del filled
    assert np.isfinite(float(copies[0].float().sum()))
