"""GPU: the index branch (write, scores, select) against its oracles.

Tolerances, u = 2^-24 the rounding of f32.
Write: a value that is quantized carries f32 roundings only: a norm's sums (8 terms a lane and a tree
of 4, twice), its root and quotient, two products, and the turn (angle in turns rounded to f32: off by
2^-26 of a turn at most, 2 pi 2^-26 < 7 u; sine and cosine 2 u; two products and a sum): below 64 u of
the row's largest value, which is also what its scale is off by, relatively. A code is off by half a
step of its own: 2^-4 of the value, 2^-10 below 2^-6.
Scores: products of E4M3 codes are exact in f32; 128 of them summed in any order, then up to 128
heads: (128 + 128) u of the sum of magnitudes at most, and a few u for the products with w and scale.
Select: whole numbers, equal.
"""

import math

import numpy as np
import pytest
import torch

from oracle import index as oindex
from tq_mla import _abi, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DIM, PAGE, ROW = 128, 64, 144


def i32(a, device):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(device)


def bf16(a, device):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(torch.bfloat16).to(device)


def host(t):
    return t.double().cpu().numpy()


def batch(rng, new, lens, spare=3):
    """Page table in no order, and sequence and position of each token (the last of each request)."""
    need = [-(-n // PAGE) for n in lens]
    order = rng.permutation(sum(need) + spare)
    table = np.full((len(lens), max(need + [1])), -1)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    seq = np.repeat(np.arange(len(lens)), new)
    pos = np.concatenate([np.arange(n - m, n) for m, n in zip(new, lens)])
    return table, seq, pos, sum(need) + spare


def check_rows(codes, scale, want):
    """Codes and scales (any leading shape) of rows whose values should be ``want``."""
    peak = np.abs(want).max(axis=-1)
    np.testing.assert_allclose(scale, peak / 448.0, rtol=64 * U + U, atol=1e-45)
    got = oindex.codes_value(codes) * scale[..., None]
    most = np.maximum(np.abs(want) * 2.0 ** -4, scale[..., None] * 2.0 ** -10) + peak[..., None] * 64 * U
    assert (np.abs(got - want) <= most).all(), np.abs(got - want).max()


# ------------------------------------------------------------------------------------- write


@pytest.mark.parametrize("new,lens,heads,rope,start,half,norm,w_type", [
    ([1], [1], 1, 0, 0, False, "none", torch.bfloat16),
    ([1], [70000], 64, 64, 0, False, "layer", torch.bfloat16),
    ([1] * 33, list(range(90, 123)), 32, 128, 0, True, "rms", torch.float32),
    ([3, 1, 200], [3, 65, 4001], 5, 16, 112, False, "rms", torch.bfloat16),
    ([77, 2], [1000, 130000], 128, 64, 64, True, "layer", torch.float32),
    ([300], [300], 8, 32, 48, True, "none", torch.bfloat16),
    ([129, 131], [129, 2 ** 20], 16, 48, 8, False, "layer", torch.bfloat16)])
def test_write(cuda_device, new, lens, heads, rope, start, half, norm, w_type):
    rng = np.random.default_rng(heads + rope)
    slim = [min(n, 4096) for n in lens]              # pages of far positions alone are not held
    table, seq, pos, pages = batch(rng, new, slim)
    pos = pos + np.repeat(np.array(lens) - np.array(slim), new) // PAGE * PAGE
    far = max(-(-n // PAGE) for n in lens)
    wide = np.full((len(lens), far), -1)
    for s, (n, m) in enumerate(zip(lens, slim)):
        shift = (n - m) // PAGE
        wide[s, shift:shift + table.shape[1]] = table[s][:far - shift]
    t = sum(new)
    q, k = bf16(rng.standard_normal((t, heads, DIM)) * 3, cuda_device), bf16(rng.standard_normal((t, DIM)) + 0.4, cuda_device)
    w = torch.from_numpy(rng.standard_normal((t, heads)).astype(np.float32)).to(cuda_device).to(w_type)
    weight = bf16(1 + 0.3 * rng.standard_normal(DIM), cuda_device) if norm != "none" else None
    bias = bf16(0.2 * rng.standard_normal(DIM), cuda_device) if norm == "layer" else None
    freq, mscale = None, 1.0
    if rope:
        freq, mscale = ops.rope_frequencies(rope, 10000.0, factor=8.0, original=8192)
        freq = freq.float().to(cuda_device)
    kv = torch.full((pages, PAGE, ROW), 0x5A, dtype=torch.uint8, device=cuda_device)
    flags = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    q_out, w_out = ops.index_write(q, k, w, i32(wide, cuda_device), i32(seq, cuda_device), i32(pos, cuda_device), kv,
                                   scale=0.25, norm_weight=weight, norm_bias=bias, freq=freq, rope_start=start,
                                   rope_half=half, rope_mscale=mscale, flags=flags)
    torch.cuda.synchronize()
    want_k, want_q = host(k), host(q)
    if norm != "none":
        want_k = oindex.normalised(want_k, host(weight), None if bias is None else host(bias), 1e-6)
    if rope:
        f = host(freq)
        want_k = oindex.turned(want_k, pos, f, start, half, mscale)
        want_q = oindex.turned(want_q, pos, f, start, half, mscale)
    rows, bad = oindex.slots(wide, seq, pos, pages)
    assert bad == 0 and int(flags) == 0
    flat = kv.view(-1, ROW).cpu().numpy()
    got = flat[rows]
    check_rows(got[:, :DIM], np.ascontiguousarray(got[:, 128:132]).view(np.float32)[:, 0].astype(np.float64), want_k)
    others = np.ones(len(flat), dtype=bool)
    others[rows] = False
    assert (flat[others] == 0x5A).all() and (flat[:, 132:] == 0x5A).all()
    scale = np.abs(want_q).max(axis=-1) / 448.0
    check_rows(q_out.cpu().numpy(), scale, want_q)
    np.testing.assert_allclose(host(w_out), host(w) * 0.25 * scale, rtol=64 * U + 3 * U, atol=1e-45)


def test_write_of_padded_strides_and_keys_alone(cuda_device):
    rng = np.random.default_rng(3)
    table, seq, pos, pages = batch(rng, [5, 9], [70, 200])
    t, h = 14, 6
    wide_q = bf16(rng.standard_normal((t, h + 2, 2 * DIM)), cuda_device)
    wide_k = bf16(rng.standard_normal((t, 3 * DIM)), cuda_device)
    q, k = wide_q[:, 1:h + 1, DIM:], wide_k[:, DIM:2 * DIM]
    w = bf16(rng.standard_normal((t, h)), cuda_device)
    ints = (i32(table, cuda_device), i32(seq, cuda_device), i32(pos, cuda_device))
    pools = [torch.zeros((pages, PAGE, r), dtype=torch.uint8, device=cuda_device) for r in (144, 160, 144)]
    a = ops.index_write(q, k, w, *ints, pools[0])
    b = ops.index_write(q.contiguous(), k.contiguous(), w, *ints, pools[1])
    assert ops.index_write(None, k, None, *ints, pools[2]) == (None, None)
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[0], pools[1][..., :144])
    check_rows(a[0].cpu().numpy(), np.abs(host(q)).max(axis=-1) / 448.0, host(q))


def test_write_skips_rows_without_a_place(cuda_device):
    rng = np.random.default_rng(4)
    table = np.array([[0, 1], [2, 77], [-5, 3]])
    seq = np.array([0, -1, 3, 1, 1, 2, 2, 0])
    pos = np.array([127, 0, 0, 64, 200, 1, 64, -1])
    k = bf16(rng.standard_normal((8, DIM)), cuda_device)
    for rows, want in (([0, 6], 0), ([1], 4), ([2], 4), ([3], 2), ([4], 8), ([5], 2), ([7], 8), (range(8), 14)):
        rows = np.array(list(rows))
        kv = torch.zeros((4, PAGE, ROW), dtype=torch.uint8, device=cuda_device)
        flags = torch.zeros(1, dtype=torch.int32, device=cuda_device)
        q = bf16(rng.standard_normal((len(rows), 3, DIM)), cuda_device)
        w = bf16(rng.standard_normal((len(rows), 3)), cuda_device)
        q_out, _ = ops.index_write(q, k[rows].contiguous(), w, i32(table, cuda_device), i32(seq[rows], cuda_device),
                                   i32(pos[rows], cuda_device), kv, flags=flags)
        torch.cuda.synchronize()
        at, bad = oindex.slots(table, seq[rows], pos[rows], 4)
        assert bad == want and int(flags) == want
        touched = (kv.view(-1, ROW) != 0).any(dim=1).nonzero().flatten().tolist()
        assert touched == sorted(at[at >= 0].tolist())
        check_rows(q_out.cpu().numpy(), np.abs(host(q)).max(axis=-1) / 448.0, host(q))


def test_write_of_rows_that_are_not_finite_zero_or_tiny(cuda_device):
    rows = torch.zeros((5, DIM), dtype=torch.bfloat16, device=cuda_device)
    rows[0, 5] = math.nan
    rows[1, 7], rows[1, 8] = math.inf, -3.0
    rows[2] = 2.0 ** -130
    rows[3, 100] = -0.0
    rows[4] = 1.0
    table = i32([[0]], cuda_device)
    kv = torch.full((1, PAGE, ROW), 9, dtype=torch.uint8, device=cuda_device)
    w = torch.ones((5, 1), dtype=torch.float32, device=cuda_device)
    q_out, w_out = ops.index_write(rows[:, None], rows, w, table, i32([0] * 5, cuda_device), i32(range(5), cuda_device), kv)
    torch.cuda.synchronize()
    codes, scale = kv[0, :5, :DIM].cpu().numpy(), kv.view(torch.float32)[0, :5, 32].cpu().numpy()
    assert np.array_equal(codes, q_out[:, 0].cpu().numpy())
    assert np.array_equal(scale, w_out[:, 0].cpu().numpy(), equal_nan=True)
    assert np.isnan(scale[0]) and (codes[0] == 0x7F).all()
    assert np.isinf(scale[1]) and codes[1, 7] == 0x7F and (codes[1, 9:] == 0).all()
    assert scale[2] > 0 and (codes[2] == codes[2, 0]).all()
    assert abs(oindex.codes_value(codes[2])[0] * float(scale[2]) - 2.0 ** -130) <= 2.0 ** -134
    assert scale[3] == 0 and (codes[3] == 0).all()
    assert (oindex.codes_value(codes[4]) == 448).all()


# ------------------------------------------------------------------------------------- scores


def index_pool(rng, pages, device, row=ROW, nan_rows=()):
    codes = rng.integers(0, 256, (pages * PAGE, DIM)).astype(np.uint8)
    codes[(codes & 0x7F) == 0x7F] = 0x41
    rows = np.full((pages * PAGE, row), 0xA7, dtype=np.uint8)
    rows[:, :DIM] = codes
    rows[:, DIM:DIM + 4] = np.exp(rng.standard_normal(pages * PAGE)).astype(np.float32)[:, None].view(np.uint8)
    return rows, torch.from_numpy(rows).to(device).view(pages, PAGE, row)


def queries(rng, tokens, heads, device):
    codes = rng.integers(0, 256, (tokens, heads, DIM)).astype(np.uint8)
    codes[(codes & 0x7F) == 0x7F] = 0x3C
    w = (rng.standard_normal((tokens, heads)) * 0.01).astype(np.float32)
    return codes, w, torch.from_numpy(codes).to(device), torch.from_numpy(w).to(device)


def check_scores(device, rng, new, lens, heads, columns=None, row=ROW, padded=0, table=None, seq=None, pos=None,
                 kv_len=None, want_flags=0):
    made = batch(rng, new, lens)
    table = made[0] if table is None else table
    seq, pos = (made[1] if seq is None else seq), (made[2] if pos is None else pos)
    kv_len = np.array(lens) if kv_len is None else kv_len
    t, pages = len(seq), made[3]
    rows, kv = index_pool(rng, pages, device, row)
    codes, w, d_codes, d_w = queries(rng, t, heads, device)
    columns = PAGE * table.shape[1] if columns is None else columns
    whole = torch.full((t, columns + padded), 7.25, dtype=torch.float32, device=device)
    out = whole[:, :columns]
    flags = torch.zeros(1, dtype=torch.int32, device=device)
    ops.index_scores(d_codes, d_w, kv, i32(table, device), i32(seq, device), i32(pos, device), i32(kv_len, device),
                     scores=out, flags=flags)
    torch.cuda.synchronize()
    want, mass = oindex.scores(codes, w, rows, table, seq, pos, kv_len, columns, np.full((t, columns), 7.25))
    got = host(out)
    seen = np.arange(columns)[None] < oindex.sees(seq, pos, kv_len, min(columns, PAGE * table.shape[1]))[:, None]
    assert (got[~seen] == 7.25).all() and (whole[:, columns:] == 7.25).all()
    err = np.abs(got - want)
    assert (err <= 260 * U * mass).all(), (err / np.maximum(mass, 1e-30)).max() / U
    assert int(flags) == want_flags


@pytest.mark.parametrize("new,lens,heads", [
    ([1], [1], 64), ([1], [63], 16), ([1], [64], 8), ([1], [65], 128), ([1], [8193], 64),
    ([1] * 9, [1, 5, 64, 127, 128, 129, 700, 3000, 2], 64),
    ([2, 4, 1, 3, 2], [300, 4, 129, 1000, 64], 48),
    ([100], [100], 64), ([257], [700], 32), ([33, 1, 70], [33, 2000, 1111], 16), ([40], [513], 8),
    ([31, 1, 17], [900, 77, 400], 24), ([19, 19], [129, 1300], 120), ([9, 3], [258, 3], 104), ([130], [400], 56)])
def test_scores(cuda_device, new, lens, heads):
    check_scores(cuda_device, np.random.default_rng(sum(lens)), new, lens, heads)


def test_scores_of_padded_rows_and_odd_columns(cuda_device):
    rng = np.random.default_rng(8)
    check_scores(cuda_device, rng, [3, 50], [400, 333], 64, columns=401, row=160, padded=5)
    check_scores(cuda_device, rng, [1, 1], [400, 333], 32, columns=333, want_flags=_abi.DEV_WORK_OVERFLOW)


def test_scores_of_tokens_out_of_order(cuda_device):
    """Sequences that alternate, positions that fall, tokens without a sequence or without rows."""
    rng = np.random.default_rng(9)
    seq = np.array([0, 1, 0, 1, 1, 1, -1, 2, 2, 3, 0, 0, -7, -1])
    pos = np.array([199, 3, 0, 640, 20, 700, 5, 0, -1, 10, 500, 100, 9, 0])
    kv_len = np.array([200, 701, 0])
    check_scores(cuda_device, rng, [1, 1, 1], [200, 701, 64], 64, seq=seq, pos=pos, kv_len=kv_len,
                 want_flags=_abi.DEV_SEQ_RANGE)


def test_scores_of_bad_tables(cuda_device):
    rng = np.random.default_rng(10)
    table, _, _, pages = batch(rng, [1, 1], [500, 300])
    broken = table.copy()
    broken[0, 2], broken[1, 0], broken[0, 7] = pages, -3, 2 ** 31 - 1
    check_scores(cuda_device, np.random.default_rng(11), [1, 1], [500, 300], 32, table=broken, want_flags=_abi.DEV_PAGE_RANGE)
    check_scores(cuda_device, np.random.default_rng(12), [1, 1], [500, 300], 32, columns=700, kv_len=np.array([500, 9000]),
                 pos=np.array([499, 8000]),      # the columns behind the second sequence's pages hold -1
                 want_flags=_abi.DEV_TABLE_SHORT | _abi.DEV_PAGE_RANGE)


def test_scores_of_rows_that_are_not_finite(cuda_device):
    """A NaN or infinite scale, or NaN codes, reach the scores that use them and no others; rows behind
    the last one that a token sees may hold anything."""
    rng = np.random.default_rng(13)
    table, seq, pos, pages = batch(rng, [4], [300])
    rows, kv = index_pool(rng, pages, cuda_device)
    at = lambda n: int(table[0, n // PAGE]) * PAGE + n % PAGE  # noqa: E731
    flat = kv.view(-1, ROW)
    flat[at(17), :DIM] = 0x7F
    flat.view(torch.float32)[at(40), 32] = math.nan
    flat.view(torch.float32)[at(150), 32] = math.inf
    for n in range(300, 320):
        flat[at(n)] = 0xFF
    codes, w, d_codes, d_w = queries(rng, 4, 64, cuda_device)
    d_codes[2, 5, 9] = 0x7F
    d_w[3, 1] = math.nan
    out = ops.index_scores(d_codes, d_w, kv, i32(table, cuda_device), i32(seq, cuda_device), i32(pos, cuda_device), i32([300], cuda_device))
    got = host(out)
    want, mass = oindex.scores(codes, w, rows, table, seq, pos, np.array([300]), out.shape[1], np.full(out.shape, -np.inf))
    seen = np.arange(out.shape[1])[None] <= pos[:, None]
    assert np.isneginf(got[~seen]).all()
    sick = np.zeros(out.shape, dtype=bool)
    sick[:, [17, 40]] = True
    sick[2:] = True
    assert np.isnan(got[sick & seen]).all()
    assert np.isinf(got[:2, 150]).all()
    sick[:, 150] = True
    well = ~sick & seen
    assert (np.abs(got - want)[well] <= (260 * U * mass)[well]).all()


# ------------------------------------------------------------------------------------- select


def check_select(device, score, seq, pos, kv_len, k, table=None, first=0, last=0, want_flags=0, d_score=None):
    flags = torch.zeros(1, dtype=torch.int32, device=device)
    if d_score is None:
        d_score = torch.from_numpy(np.ascontiguousarray(score, dtype=np.float32)).to(device)
    idx, length = ops.index_select(d_score, i32(seq, device), i32(pos, device), i32(kv_len, device), k, flags=flags,
                                   page_table=None if table is None else i32(table, device), keep_first=first, keep_last=last)
    torch.cuda.synchronize()
    want, want_len = oindex.select(score, seq, pos, kv_len, k, table, first, last)
    np.testing.assert_array_equal(length.cpu().numpy(), want_len)
    np.testing.assert_array_equal(idx.cpu().numpy(), want)
    assert int(flags) == want_flags


VALUES = ["normal", "coarse", "equal", "zeros", "tiny", "wide", "one high", "falling", "rising", "masked", "clusters", "runs high",
          "runs low", "two values"]


def values(kind, rng, t, n):
    v = rng.standard_normal((t, n)).astype(np.float32)
    if kind == "coarse":
        v = np.round(v * 4) / 4
    if kind == "equal":
        v = np.full_like(v, -2.5)
    if kind == "zeros":
        v = np.where(rng.random((t, n)) < 0.5, 0.0, -0.0).astype(np.float32)
        v[rng.random((t, n)) < 0.02] = -1.0
    if kind == "tiny":
        v = (v * 1e-41).astype(np.float32)
    if kind == "wide":
        v = (np.sign(v) * np.exp(rng.uniform(-80, 80, (t, n)))).astype(np.float32)
    if kind == "one high":
        v[:, n // 3] = 3e38
        v[:, n // 2] = np.inf
    if kind == "falling":
        v = -np.sort(-v, axis=1)
    if kind == "rising":
        v = np.sort(v, axis=1)
    if kind == "masked":
        v[rng.random((t, n)) < 0.9] = -np.inf
        v[rng.random((t, n)) < 0.03] = np.nan
        v[rng.random((t, n)) < 0.03] = np.finfo(np.float32).min
        v[0] = -np.inf
    if kind in ("runs high", "runs low"):       # evenly spaced neighbours unlike the rest
        for part in range(512):
            at = part * max(n - 8, 0) // 512
            v[:, at:at + 8] += 20 if kind == "runs high" else -20
    if kind == "two values":
        v = np.where(rng.random((t, n)) < 0.5, 3.0, -1.5).astype(np.float32)
    if kind == "clusters":
        v = (np.where(rng.random((t, n)) < 0.97, 1.0, 8.0) + v * 1e-6).astype(np.float32)
    return v


@pytest.mark.parametrize("kind", VALUES)
@pytest.mark.parametrize("n,k", [(1, 1), (5, 9), (129, 128), (1000, 7), (4099, 2051), (20011, 2048), (70001, 301)])
def test_select(cuda_device, kind, n, k):
    rng = np.random.default_rng(n + k)
    t = 3
    check_select(cuda_device, values(kind, rng, t, n), np.arange(t), np.full(t, n - 1), np.full(t, n), k)


@pytest.mark.parametrize("kind", VALUES)
@pytest.mark.parametrize("n,k,first,last", [(1, 1, 0, 0), (64, 2, 1, 1), (65, 1, 0, 1), (1000, 5, 0, 0), (9001, 40, 2, 3),
                                            (70001, 100, 1, 1), (131072, 2051, 0, 1)])
def test_select_pages(cuda_device, kind, n, k, first, last):
    rng = np.random.default_rng(n + k)
    t = 2
    columns = -(-n // PAGE)
    table = rng.permutation(t * columns).reshape(t, columns)
    check_select(cuda_device, values(kind, rng, t, n), np.arange(t), np.full(t, n - 1), np.full(t, n), k, table, first, last)


def test_select_keeps_the_first_and_the_last(cuda_device):
    rng = np.random.default_rng(20)
    score = values("masked", rng, 4, 700)
    score[1, :3], score[2, 690:] = np.nan, -np.inf
    for k, first, last in ((10, 4, 6), (10, 10, 0), (10, 0, 10), (300, 3, 5), (700, 1, 1), (2000, 900, 900)):
        check_select(cuda_device, score, np.arange(4), np.array([699, 300, 699, 4]), np.full(4, 700), k, None, first, last)


def test_select_of_what_each_token_sees(cuda_device):
    """Tokens that see nothing, one row, part of a page; scores behind it are never read as scores; no
    sequence; more rows than columns or than the page table holds."""
    rng = np.random.default_rng(21)
    seq = np.array([0, 1, 2, 2, 0, 1, -1, 3, 0])
    pos = np.array([-1, 0, 63, 64, 199, 900, 3, 3, 10 ** 9])
    kv_len = np.array([200, 150, 400])
    score = values("normal", rng, 9, 400)
    n = oindex.sees(seq, pos, kv_len, 400)
    score[np.arange(400)[None] >= n[:, None]] = np.inf
    table = rng.permutation(21).reshape(3, 7)
    for k in (1, 64, 130):
        check_select(cuda_device, score, seq, pos, kv_len, k, want_flags=_abi.DEV_SEQ_RANGE)
        check_select(cuda_device, score, seq, pos, kv_len, k, table, want_flags=_abi.DEV_SEQ_RANGE)
    wide = values("normal", rng, 2, 500)
    check_select(cuda_device, wide, np.array([0, 1]), np.array([600, 20]), np.array([601, 21]), 9, want_flags=_abi.DEV_WORK_OVERFLOW)
    check_select(cuda_device, wide, np.array([0, 1]), np.array([499, 20]), np.array([500, 21]), 9, table[:2], want_flags=_abi.DEV_TABLE_SHORT)


def test_select_of_padded_and_unaligned_rows(cuda_device):
    rng = np.random.default_rng(22)
    for width, start, n in ((1003, 1, 997), (1003, 3, 1000), (1024, 4, 777)):
        whole = torch.from_numpy(values("normal", rng, 5, width)).to(cuda_device)
        part = whole[:, start:start + n]
        check_select(cuda_device, part.cpu().numpy(), np.zeros(5, int), np.arange(n - 5, n), np.array([n]), 100, d_score=part)
        table = rng.permutation(16)[None]
        check_select(cuda_device, part.cpu().numpy(), np.zeros(5, int), np.arange(n - 5, n), np.array([n]), 7, table, d_score=part)


def test_select_of_many_rows(cuda_device):
    rng = np.random.default_rng(23)
    t, n = 700, 3001
    check_select(cuda_device, values("normal", rng, t, n), np.zeros(t, int), np.arange(n - t, n), np.array([n]), 512)


@pytest.mark.parametrize("kind", VALUES)
@pytest.mark.parametrize("t,n,k", [(40, 40003, 301), (148, 16390, 2051), (149, 16390, 60), (500, 1503, 200), (150, 2049, 9)])
def test_select_of_rows_that_fill_the_card(cuda_device, kind, t, n, k):
    """About as many rows as there are SMs, and many short ones."""
    rng = np.random.default_rng(t + k)
    score = values(kind, rng, t, n)
    last = np.arange(n - t, n)
    check_select(cuda_device, score, np.zeros(t, int), last, np.array([n]), k)
    check_select(cuda_device, score, np.zeros(t, int), last, np.array([n]), k, None, 3, k // 2)


@pytest.mark.parametrize("kind", ["normal", "equal", "runs low"])
def test_select_of_the_longest_rows(cuda_device, kind):
    rng = np.random.default_rng(24)
    n = 1 << 20
    score = values(kind, rng, 1, n)
    check_select(cuda_device, score, np.array([0]), np.array([n - 1]), np.array([n]), 2051)
    check_select(cuda_device, score, np.array([0]), np.array([n - 1]), np.array([n]), 2051, rng.permutation(n // PAGE)[None], 1, 2)


def test_select_of_no_columns(cuda_device):
    score = torch.zeros((2, 0), device=cuda_device)
    idx, length = ops.index_select(score, i32([0, 1], cuda_device), i32([0, 0], cuda_device), i32([0, 0], cuda_device), 3)
    assert (idx == -1).all() and (length == 0).all()
