"""Index operators where byte offsets pass 32 bits, and with many tokens: the same bits as the same
work at small offsets."""

import numpy as np
import pytest
import torch

from oracle import index as oindex
from test_gpu_index import DIM, PAGE, batch, check_scores, i32, index_pool, queries
from tq_mla import ops

pytestmark = pytest.mark.gpu
ROW = 144


def test_cache_past_4_gib(cuda_device):
    rng = np.random.default_rng(1)
    table, seq, pos, pages = batch(rng, [2, 3], [700, 130])
    most = 2 ** 32 // (PAGE * ROW) + 70
    far = np.where(table >= 0, table + most - pages, -1)
    assert (most - pages) * PAGE * ROW >= 2 ** 32
    rows, near_kv = index_pool(rng, pages, cuda_device)
    far_kv = torch.zeros((most, PAGE, ROW), dtype=torch.uint8, device=cuda_device)
    far_kv[most - pages:] = near_kv
    q = torch.randn((5, 64, DIM), device=cuda_device).bfloat16()
    k = torch.randn((5, DIM), device=cuda_device).bfloat16()
    w = torch.randn((5, 64), device=cuda_device)
    d_seq, d_pos, kv_len = i32(seq, cuda_device), i32(pos, cuda_device), i32([700, 130], cuda_device)
    found = []
    for kv, t in ((near_kv, table), (far_kv, far)):
        t = i32(t, cuda_device)
        codes, w8 = ops.index_write(q, k, w, t, d_seq, d_pos, kv)
        scores = ops.index_scores(codes, w8, kv, t, d_seq, d_pos, kv_len)
        idx, length = ops.index_select(scores, d_seq, d_pos, kv_len, 4, page_table=t, keep_first=1)
        found.append((scores, idx, length))
    torch.cuda.synchronize()
    (a, i, n), (b, j, m) = found
    assert torch.equal(a, b) and torch.equal(n, m) and torch.equal(torch.where(i >= 0, i + most - pages, i), j)
    assert torch.equal(far_kv[most - pages:], near_kv) and not far_kv[:most - pages].any()


def test_queries_past_4_gib(cuda_device):
    t, heads = 2 ** 32 // (128 * DIM * 2) + 3, 128
    q = torch.zeros((t, heads, DIM), dtype=torch.bfloat16, device=cuda_device)
    w = torch.zeros((t, heads), device=cuda_device)
    k = torch.zeros((t, DIM), dtype=torch.bfloat16, device=cuda_device)
    for x in (q, w, k):
        x[-3:] = torch.randn(x[-3:].shape, device=cuda_device).to(x.dtype)
    seq, pos = torch.full((t,), -1, dtype=torch.int32, device=cuda_device), torch.zeros(t, dtype=torch.int32, device=cuda_device)
    seq[-3:], pos[-3:] = 0, i32([5, 6, 7], cuda_device)
    table, freq = i32([[1]], cuda_device), torch.rand(32, device=cuda_device)
    kvs = [torch.zeros((2, PAGE, ROW), dtype=torch.uint8, device=cuda_device) for _ in range(2)]
    codes, w8 = ops.index_write(q, k, w, table, seq, pos, kvs[0], freq=freq)
    want, want8 = ops.index_write(q[-3:], k[-3:], w[-3:], table, seq[-3:], pos[-3:], kvs[1], freq=freq)
    assert torch.equal(codes[-3:], want) and torch.equal(w8[-3:], want8) and torch.equal(*kvs) and want.any()
    assert not codes[:-3].any() and not w8[:-3].any()


def test_scores_past_4_gib(cuda_device):
    """Rows of 2^20 columns, read and written at the end of more than 4 GiB."""
    rng = np.random.default_rng(2)
    t, n = 1030, 2 ** 20
    rows, kv = index_pool(rng, 8, cuda_device)
    _, _, codes, w = queries(rng, t, 16, cuda_device)
    table, kv_len = i32(rng.permutation(8)[None], cuda_device), i32([500], cuda_device)
    seq = torch.zeros(t, dtype=torch.int32, device=cuda_device)
    pos = torch.full((t,), -1, dtype=torch.int32, device=cuda_device)
    pos[-4:] = i32([0, 130, 400, 499], cuda_device)
    scores = torch.full((t, n), -np.inf, device=cuda_device)
    ops.index_scores(codes, w, kv, table, seq, pos, kv_len, scores=scores)
    want = ops.index_scores(codes[-4:], w[-4:], kv, table, seq[-4:], pos[-4:], kv_len)
    assert torch.equal(scores[-4:, :512], want) and torch.isneginf(scores[-4:, 512:]).all() and torch.isneginf(scores[:8]).all()
    scores[-4:] = torch.randn((4, n), device=cuda_device)
    pos[-4:] = i32([n - 1, n - 70, 5, n // 2], cuda_device)
    kv_len = i32([n], cuda_device)
    pages = torch.arange(n // PAGE, dtype=torch.int32, device=cuda_device)[None]
    for page_table in (None, pages):
        idx, length = ops.index_select(scores, seq, pos, kv_len, 100, page_table=page_table)
        near, near_len = ops.index_select(scores[-4:].clone(), seq[-4:], pos[-4:], kv_len, 100, page_table=page_table)
        assert torch.equal(idx[-4:], near) and torch.equal(length[-4:], near_len)
        assert (idx[:-4] == -1).all() and (length[:-4] == 0).all()
        want, want_len = oindex.select(scores[-4:].cpu().numpy(), np.zeros(4, int), pos[-4:].cpu().numpy(), np.array([n]), 100,
                                       None if page_table is None else pages.cpu().numpy())
        np.testing.assert_array_equal(near.cpu().numpy(), want)
        np.testing.assert_array_equal(near_len.cpu().numpy(), want_len)


@pytest.mark.parametrize("heads", [8, 16])
def test_many_tokens(cuda_device, heads):
    """More tokens than are looked up once, in runs of one to ninety."""
    rng = np.random.default_rng(heads)
    new = rng.integers(0, 90, 800)
    lens = new + rng.integers(0, 40, 800)
    check_scores(cuda_device, rng, new.tolist(), lens.tolist(), heads)
    t = int(new.sum())
    made, seq, pos, _ = batch(rng, new.tolist(), lens.tolist())
    score = rng.standard_normal((t, 64 * made.shape[1])).astype(np.float32)
    idx, length = ops.index_select(torch.from_numpy(score).to(cuda_device), i32(seq, cuda_device), i32(pos, cuda_device),
                                   i32(lens, cuda_device), 17)
    want, want_len = oindex.select(score, seq, pos, lens, 17)
    np.testing.assert_array_equal(idx.cpu().numpy(), want)
    np.testing.assert_array_equal(length.cpu().numpy(), want_len)
