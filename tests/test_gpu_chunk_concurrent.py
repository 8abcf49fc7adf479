"""GPU: chunk attention calls on several streams at once, launched and replayed, beside norms and step
plans: CTAs of different kernels come and go on the same SMs, and the two CTAs of a pair start at
different times. Every call gives the bits that it gives alone, and every call ends."""

import numpy as np
import pytest
import torch

from test_gpu_chunk import Case, i32
from test_gpu_chunk_order import LEVELS, growing
from tq_mla import ops

pytestmark = pytest.mark.gpu
ROUNDS = 5000


def test_calls_on_many_streams_at_once(cuda_device):
    dev = cuda_device
    cases = [Case(dev, 2, [200, 3, 700], [700, 2000, 0], heads=16, seed=1),
             growing(dev, 0, [300, 512], [1000, 0], LEVELS["every tile"], 8, seed=2),
             growing(dev, 1, [1, 40, 600], [3000, 100, 900], LEVELS["every tile"], 16, seed=3),
             Case(dev, 2, [24], [100], heads=16, seed=4)]
    launches = [c.launch() for c in cases]
    rng = np.random.default_rng(5)
    y, residual = (torch.from_numpy(rng.standard_normal((1021, 5192)).astype(np.float32)).to(dev).to(torch.bfloat16)
                   for _ in range(2))
    norm = ops.BlockNorm(y, residual, torch.empty_like(residual),
                         post_weight=torch.ones(5192, dtype=torch.bfloat16, device=dev))
    plan = ops.StepPlan(i32(np.full(64, 100), dev), i32(np.full(64, 30), dev), i32(np.zeros((64, 9)), dev),
                        i32(np.arange(500), dev), i32([500], dev), tokens=2000)
    for call in launches + [norm, plan]:
        call()
    torch.cuda.synchronize()
    want = [(c.out.clone(), c.lse.clone()) for c in cases]
    want_small = [t.clone() for t in (norm.out, *plan.tables)]
    streams = [torch.cuda.Stream() for _ in cases]
    extra = torch.cuda.Stream()
    graphs = []
    for launch, stream in zip(launches, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            launch()
        graphs.append(graph)
    torch.cuda.synchronize()
    for k in range(ROUNDS):
        if k % 50 == 0:
            for c in cases:
                c.out.fill_(7.0)
                c.lse.fill_(7.0)
            torch.cuda.synchronize()
        for _ in range(int(rng.integers(1, 5))):
            for i in rng.permutation(len(cases)):
                if rng.random() < 0.5:
                    launches[i](streams[i])
                else:
                    with torch.cuda.stream(streams[i]):
                        graphs[i].replay()
            norm(extra)
            plan(stream=extra)
        torch.cuda.synchronize()
        if k % 10 == 0 or k == ROUNDS - 1:
            # every stream has made at least one call since the outputs were cleared
            for c, launch, (out, lse) in zip(cases, launches, want):
                assert launch.device_error() == 0
                assert torch.equal(c.out, out) and torch.equal(c.lse, lse)
            for got, ref in zip((norm.out, *plan.tables), want_small):
                assert torch.equal(got, ref)
    del graph
    graphs.clear()
