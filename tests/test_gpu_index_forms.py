"""GPU: the forms of the index kernels that sizes choose: every head count of the scores, parts of a token's
heads in the write, pages of many full rows and of the longest ones in the select. Tolerances: see
``test_gpu_index``."""

import numpy as np
import pytest
import torch

from oracle import index as oindex
from test_gpu_index import DIM, PAGE, ROW, U, batch, bf16, check_rows, check_scores, check_select, host, i32, index_pool, queries, values
from tq_mla import ops

pytestmark = pytest.mark.gpu

# The tokens of a step are 256 / heads, 16 at most.
HEADS = [8, 16, 24, 32, 40, 48, 56, 64, 72, 80, 88, 96, 104, 112, 120, 128]


def a_step(heads):
    return min(16, 256 // heads)


# ------------------------------------------------------------------------------------- scores


@pytest.mark.parametrize("heads", HEADS)
def test_scores_of_single_tokens(cuda_device, heads):
    """Several tiles a step, a last step that is not full, runs that end in their first tile."""
    check_scores(cuda_device, np.random.default_rng(heads), [1] * 9, [1, 300, 1025, 640, 129, 1, 2000, 513, 64], heads)


@pytest.mark.parametrize("heads", HEADS)
def test_scores_of_two_and_three_tokens(cuda_device, heads):
    check_scores(cuda_device, np.random.default_rng(heads), [2, 3, 2, 3, 1], [700, 1300, 2, 333, 129], heads)


@pytest.mark.parametrize("heads", HEADS)
def test_scores_of_runs_about_a_step(cuda_device, heads):
    """One token more than a step holds, which leaves warps without a token; one less; a whole group and one
    more; with few tiles and many."""
    n = a_step(heads)
    new = [n + 1, n, 2 * n, 2 * n + 1, max(1, n - 1), 2 * n - 1]
    check_scores(cuda_device, np.random.default_rng(heads), new, [900, 1500, 2 * n, 400, 130, 1100], heads)
    check_scores(cuda_device, np.random.default_rng(heads + 1), [n + 1], [n + 1], heads)
    check_scores(cuda_device, np.random.default_rng(heads + 2), [n + 1], [4000], heads)


@pytest.mark.parametrize("heads", HEADS)
def test_scores_of_many_units(cuda_device, heads):
    """Blocks that walk several runs, with tiles of a share that starts and ends inside them."""
    rng = np.random.default_rng(heads)
    new = rng.integers(1, 24, 30)
    check_scores(cuda_device, rng, new.tolist(), (new + rng.integers(0, 500, 30)).tolist(), heads)


@pytest.mark.parametrize("heads", [1, 4, 12, 33])
def test_scores_of_heads_that_are_filled_up(cuda_device, heads):
    """Heads filled up to a multiple of 8 with queries and weights of zero change no score."""
    rng = np.random.default_rng(heads)
    table, seq, pos, pages = batch(rng, [2, 1, 20], [300, 65, 130])
    rows, kv = index_pool(rng, pages, cuda_device)
    t, full = len(seq), -(-heads // 8) * 8
    q = torch.zeros((t, full, DIM), dtype=torch.bfloat16, device=cuda_device)
    w = torch.zeros((t, full), device=cuda_device)
    q[:, :heads] = bf16(rng.standard_normal((t, heads, DIM)), cuda_device)
    w[:, :heads] = torch.from_numpy(rng.standard_normal((t, heads)).astype(np.float32))
    where = (i32(table, cuda_device), i32(seq, cuda_device), i32(pos, cuda_device))
    written = torch.zeros_like(kv)
    codes, w8 = ops.index_write(q, q[:, 0].contiguous(), w, *where, written)
    assert not codes[:, heads:].any() and not w8[:, heads:].any()
    scores = ops.index_scores(codes, w8, kv, *where, i32([300, 65, 130], cuda_device))
    want, mass = oindex.scores(codes[:, :heads].cpu().numpy(), host(w8[:, :heads]), rows, table, seq, pos,
                               np.array([300, 65, 130]), scores.shape[1], np.full(scores.shape, -np.inf))
    seen = np.isfinite(want)
    assert np.array_equal(np.isfinite(host(scores)), seen)
    assert (np.abs(host(scores)[seen] - want[seen]) <= 260 * U * mass[seen]).all()


@pytest.mark.parametrize("heads", [8, 16, 64, 128])
def test_scores_of_large_sums(cuda_device, heads):
    """Sums of magnitudes just below 2^127 stay finite for every key."""
    n = 200
    rng = np.random.default_rng(heads)
    table, seq, pos, pages = batch(rng, [2], [n])
    kv = torch.zeros((pages, PAGE, ROW), dtype=torch.uint8, device=cuda_device)
    kv[..., :DIM] = 0x7E                                                # 448
    kv.view(torch.float32)[..., DIM // 4] = 0.5
    codes = torch.full((2, heads, DIM), 0x7E, dtype=torch.uint8, device=cuda_device)
    dot = 448.0 * 448.0 * DIM                                           # whole numbers below 2^25: exact
    each = np.float32(2.0 ** 127 * (1 - 2.0 ** -10) / (dot * heads))
    w = torch.full((2, heads), float(each), device=cuda_device)
    w[1, 1::2] *= -1
    scores = ops.index_scores(codes, w, kv, i32(table, cuda_device), i32(seq, cuda_device), i32(pos, cuda_device), i32([n], cuda_device))
    got = host(scores)
    want = 0.5 * dot * heads * float(each)
    assert (np.abs(got[0, :n - 1] - want) <= 260 * U * want).all()
    assert (np.abs(got[1, :n]) <= 260 * U * want).all()


# ------------------------------------------------------------------------------------- write


@pytest.mark.parametrize("tokens,heads", [(3000, 30), (4400, 31), (5500, 48), (9000, 33), (2700, 100)])
@pytest.mark.parametrize("rope,half", [(0, False), (64, False), (32, True), (128, True)])
def test_write_of_many_heads_a_warp(cuda_device, tokens, heads, rope, half):
    """Eight, sixteen and thirty-two heads a warp, the last part of a token's heads not full: the bits of
    calls of few tokens, which have four a warp, and the values of the definition."""
    rng = np.random.default_rng(heads + rope)
    g = torch.Generator(device=cuda_device).manual_seed(heads)
    q = torch.randn((tokens, heads, DIM), generator=g, device=cuda_device).bfloat16()
    k = torch.randn((tokens, DIM), generator=g, device=cuda_device).bfloat16()
    w = torch.randn((tokens, heads), generator=g, device=cuda_device)
    freq = None
    if rope:
        freq = ops.rope_frequencies(rope, 10000.0)[0].float().to(cuda_device)
    pages = -(-tokens // PAGE)
    where = (i32(rng.permutation(pages)[None], cuda_device), torch.zeros(tokens, dtype=torch.int32, device=cuda_device),
             torch.arange(tokens, dtype=torch.int32, device=cuda_device))
    kw = dict(scale=0.25, freq=freq, rope_half=half, rope_start=0 if rope == 128 else 48)
    kvs = [torch.zeros((pages, PAGE, ROW), dtype=torch.uint8, device=cuda_device) for _ in range(2)]
    codes, w8 = ops.index_write(q, k, w, *where, kvs[0], **kw)
    step = 500
    assert step * heads < 65536                     # below that a warp has four
    for a in range(0, tokens, step):
        part, part_w = ops.index_write(q[a:a + step], k[a:a + step], w[a:a + step], where[0], where[1][a:a + step],
                                       where[2][a:a + step], kvs[1], **kw)
        assert torch.equal(part, codes[a:a + step]) and torch.equal(part_w, w8[a:a + step])
    assert torch.equal(*kvs)
    some = np.sort(rng.choice(tokens, 40, replace=False))
    want = host(q[some])
    if rope:
        want = oindex.turned(want, some, host(freq), kw["rope_start"], half)
    scale = np.abs(want).max(axis=-1) / 448.0
    check_rows(codes[some].cpu().numpy(), scale, want)
    np.testing.assert_allclose(host(w8[some]), host(w[some]) * 0.25 * scale, rtol=64 * U + 3 * U)


# ------------------------------------------------------------------------------------- select


@pytest.mark.parametrize("kind", ["normal", "coarse", "equal", "masked", "rising", "clusters"])
@pytest.mark.parametrize("t,n,k,first,last", [(400, 4096, 64, 1, 1), (1000, 1500, 5, 0, 0), (149, 70001, 300, 2, 1)])
def test_pages_of_more_rows_than_sms(cuda_device, kind, t, n, k, first, last):
    """A prompt's tokens: each sees one row more than the one before, the last all of them."""
    rng = np.random.default_rng(t + k)
    table = rng.permutation(-(-n // PAGE))[None]
    check_select(cuda_device, values(kind, rng, t, n), np.zeros(t, int), np.arange(n - t, n), np.array([n]), k, table, first, last)


@pytest.mark.parametrize("n,kind", [(140001, "normal"), (140001, "equal"), (140001, "masked"), (140001, "rising"),
                                    (530001, "normal"), (530001, "masked")])
def test_pages_of_many_long_rows(cuda_device, n, kind):
    """Thousands of pages a block: more rows than clusters are made for, longer than 2048 and 8192 pages."""
    t = 75
    rng = np.random.default_rng(n)
    table = rng.permutation(-(-n // PAGE))[None]
    score = values(kind, rng, t, n)
    check_select(cuda_device, score, np.zeros(t, int), np.arange(n - t, n), np.array([n]), 500, table, 1, 1)
