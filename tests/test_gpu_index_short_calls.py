"""GPU: index scores of calls that end right after they began: a tile or two a block, none in most blocks,
behind one another and beside each other."""

import numpy as np
import pytest
import torch

from test_gpu_index import batch, i32, index_pool, queries
from tq_mla import ops

pytestmark = pytest.mark.gpu


def test_short_calls_behind_and_beside_each_other(cuda_device):
    """Each of them gives the bits that it gives alone. (One to ten tiles, so that the last arrivals on a
    block's barriers come as it ends; forms of both sums and of one and two steps a tile.)"""
    rng = np.random.default_rng(1)
    calls = []
    for new, lens, heads in (([1], [1], 64), ([1], [129], 16), ([1], [1200], 128), ([3], [200], 128), ([1], [300], 24),
                             ([30], [30], 16), ([1, 1, 1], [64, 700, 3], 48), ([1], [0], 8)):
        table, seq, pos, pages = batch(rng, new, lens)
        _, kv = index_pool(rng, pages, cuda_device)
        _, _, codes, w = queries(rng, len(seq), heads, cuda_device)
        scores = torch.full((len(seq), 64 * table.shape[1]), -np.inf, device=cuda_device)
        calls.append(ops.IndexScores(codes, w, kv, i32(table, cuda_device), i32(seq, cuda_device), i32(pos, cuda_device),
                                     i32(lens, cuda_device), scores))
    flags = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    want = []
    for call in calls:
        call(flags)
        torch.cuda.synchronize()
        want.append(call.scores.clone())
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(40):
        for call in calls:
            call.scores.fill_(-np.inf)
        torch.cuda.synchronize()
        for _ in range(25):
            for i in rng.permutation(len(calls)):
                with torch.cuda.stream(streams[i]):
                    calls[i](flags)
        torch.cuda.synchronize()
        for _ in range(25):                       # one stream: each starts while the one before ends
            for i in rng.permutation(len(calls)):
                with torch.cuda.stream(streams[0]):
                    calls[i](flags)
        torch.cuda.synchronize()
        assert all(torch.equal(call.scores, x) for call, x in zip(calls, want))
    assert int(flags) == 0
