"""GPU: index scores of the longest row that can be declared, 2^31 - 1 columns: row counts that leave no
room in 31 bits for a tile's rows beside them."""

import numpy as np
import pytest
import torch

from test_gpu_index import PAGE, i32, index_pool, queries
from tq_mla import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,tokens", [(16, 1), (8, 1), (128, 3)])
def test_a_row_of_all_columns(cuda_device, heads, tokens):
    """One page, again and again in the page table: each tile's scores are the first tile's, bit for bit. The
    last token sees all rows, those before it a few (128 heads: three tokens are two steps a tile)."""
    n, tile = 2 ** 31 - 1, 2 * PAGE
    rng = np.random.default_rng(heads)
    _, kv = index_pool(rng, 1, cuda_device)
    _, _, codes, w = queries(rng, tokens, heads, cuda_device)
    table = torch.zeros((1, 2 ** 31 // PAGE), dtype=torch.int32, device=cuda_device)
    seq = torch.zeros(tokens, dtype=torch.int32, device=cuda_device)
    pos = i32(list(range(100, 99 + tokens)) + [n], cuda_device)
    flags = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    scores = torch.full((tokens, n), -np.inf, device=cuda_device)
    ops.index_scores(codes, w, kv, table, seq, pos, i32([n], cuda_device), scores=scores, flags=flags)
    want = ops.index_scores(codes, w, kv, i32([[0, 0]], cuda_device), seq, torch.clamp(pos, max=tile - 1), i32([tile], cuda_device))
    assert bool(torch.isfinite(want[-1]).all()) and int(flags) == 0
    for t in range(tokens - 1):
        assert torch.equal(scores[t, :tile], want[t]) and bool(torch.isneginf(scores[t, tile:]).all())
    whole = n // tile * tile
    for at in range(0, whole, 2 ** 28):
        part = scores[-1, at:min(whole, at + 2 ** 28)].view(-1, tile)
        assert bool((part == want[-1]).all()), at
    assert torch.equal(scores[-1, whole:], want[-1, :n - whole])
