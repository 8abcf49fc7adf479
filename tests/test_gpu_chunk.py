"""GPU: chunk attention against its float64 oracle.

Tolerances. With h = 2^-8, bf16's largest relative rounding error, an expanded key or value is off by
at most h of itself, after a sum of 512 products in f32: each of the 512 additions rounds by at most
2^-24 of a partial sum, and no partial sum exceeds sum_r |latent_r w_r|, so that sum is off by at most
512 * 2^-24 = 2^-15 of sum_r |latent_r w_r| (it matters where the sum cancels, in a row that sees one
key). FP8 rows' latent values are rounded to bf16 first, which adds h of the same sum. A score is off
by at most
d = scale * sum |q| |key error|, a softmax weight by a factor within exp(+-2d), and it is rounded
once more, as is the value. The output is then off by at most
  sum_n p_n |value error|  +  (exp(2d) - 1 + h)(1 + h) sum_n p_n |v_n|  +  half a step of its type,
lse by at most d, plus f32 terms: 2^-16 of the largest score covers sums of at most a few thousand
f32 products and the exponential's error. That is what no element may pass. Roundings are
independent, each of rms h / sqrt(3) of its value, so that over all elements the relative 2-norm
stays within 1e-2 for scores of unit spread."""

import numpy as np
import pytest
import torch

from oracle import chunk as ochunk
from oracle import fp8 as ofp8
from tq_mla import _abi, ops

pytestmark = pytest.mark.gpu
H = 2.0 ** -8
STRIDE = {0: 1024, 1: 544, 2: 1152}


def bf16(a, device):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(torch.bfloat16).to(device)


def i32(a, device):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(device)


def f64(t):
    return t.double().cpu().numpy()


class Case:
    """A seeded batch: host and device copies of everything a call takes."""

    def __init__(self, device, fmt, new, cached, heads=3, seed=0, spare=2, lead=0, tail=0, row_pad=0):
        rng = np.random.default_rng(seed + 10 * fmt)
        self.device, self.fmt, self.heads = device, fmt, heads
        dn, self.dr = (128, 64) if fmt == 2 else (256, 0)
        self.dn = self.dv = dn
        new, cached = np.array(new), np.array(cached)
        lens = new + cached
        self.seqs, self.tokens = len(new), int(new.sum()) + lead + tail
        need = -(-lens // 64)
        slots, pages = max(1, int(need.max())), int(need.sum()) + spare
        order = rng.permutation(pages)
        table = np.full((self.seqs, slots), -1)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        stride = STRIDE[fmt] + row_pad
        pool = torch.full((pages * 64, stride), 255, dtype=torch.uint8, device=device)   # NaN
        live = np.concatenate([table[s, np.arange(n) // 64] * 64 + np.arange(n) % 64
                               for s, n in enumerate(lens)]).astype(np.int64)
        live_t = torch.from_numpy(live).to(device)
        values = rng.standard_normal((len(live), 512 + self.dr)).astype(np.float32)
        if fmt == 1:
            tiles = torch.from_numpy(values).view(-1, 4, 128)
            scale = tiles.abs().amax(dim=2) / 448
            codes = (tiles / scale[:, :, None]).to(torch.float8_e4m3fn).view(-1, 512).view(torch.uint8)
            pool[live_t, :512] = codes.to(device)
            pool[live_t, 512:528] = scale.contiguous().view(torch.uint8).view(-1, 16).to(device)
        else:
            raw = torch.from_numpy(values).to(torch.bfloat16).view(torch.uint8).view(len(live), -1)
            pool[live_t, :raw.shape[1]] = raw.to(device)
        self.live = live
        self.kv = pool.view(pages, 64, stride)
        self.table = table
        self.q_start = lead + np.concatenate([[0], np.cumsum(new)])
        self.kv_len = lens
        self.q_pos = np.concatenate([np.full(lead, 5)] + [np.arange(c, c + n) for n, c in zip(new, cached)] +
                                    [np.full(tail, 5)])
        self.q = bf16(rng.standard_normal((self.tokens, heads, dn + self.dr)), device)
        self.w_uk = bf16(rng.standard_normal((heads, dn, 512)) / np.sqrt(512), device)
        self.w_uv = bf16(rng.standard_normal((heads, dn, 512)) / np.sqrt(512), device)
        self.scale = (dn + self.dr) ** -0.5
        self.max_keys = int(lens[new > 0].sum())

    def args(self):
        d = self.device
        return (self.q, self.w_uk, self.w_uv, self.kv, i32(self.table, d), i32(self.q_start, d),
                i32(self.q_pos, d), i32(self.kv_len, d))

    def launch(self, out_dtype=torch.bfloat16, lse=True, **kw):
        self.out = torch.full((self.tokens, self.heads, self.dv), 7.0, dtype=out_dtype, device=self.device)
        self.lse = torch.full((self.tokens, self.heads), 7.0, device=self.device) if lse else None
        kw.setdefault("max_keys", self.max_keys)
        return ops.MlaChunk(*self.args(), self.out, self.lse, scale=self.scale, kv_format=self.fmt, **kw)

    def rows(self):
        with np.errstate(invalid="ignore"):
            return ochunk.pool_rows(self.kv.reshape(-1, self.kv.shape[-1]).cpu().numpy(), self.fmt)

    def oracle(self):
        return ochunk.chunk_attention(f64(self.q), f64(self.w_uk), f64(self.w_uv), self.rows(), self.table,
                                      self.q_start, self.q_pos, self.kv_len, scale=self.scale)

    def bounds(self):
        """Per element: the largest error of out before its own rounding, and of lse."""
        q, uk, uv, rows = np.abs(f64(self.q)), f64(self.w_uk), f64(self.w_uv), self.rows()
        off_out = np.zeros((self.tokens, self.heads, self.dv))
        off_lse = np.zeros((self.tokens, self.heads))
        signed = f64(self.q)
        latent_off = H if self.fmt == 1 else 0.0
        for s in range(self.seqs):
            b, e, n = int(self.q_start[s]), int(self.q_start[s + 1]), int(self.kv_len[s])
            if e <= b or n <= 0:
                continue
            pos = np.arange(n)
            page = self.table[s, np.minimum(pos // 64, self.table.shape[1] - 1)]
            known = (page >= 0) & (page < self.kv.shape[0])
            kv = np.where(known[:, None], rows[np.where(known, page, 0) * 64 + pos % 64], 0.0)
            kv = np.where(np.isfinite(kv).all(axis=1)[:, None], kv, 0.0)
            lat = kv[:, :512]
            hidden = pos[None] >= np.minimum(n, self.q_pos[b:e, None] + 1)
            for h in range(self.heads):
                k, v = lat @ uk[h].T, lat @ uv[h].T
                before = (1 + H) * (latent_off + 2.0 ** -15)
                k_off = H * np.abs(k) + before * (np.abs(lat) @ np.abs(uk[h]).T)
                v_off = H * np.abs(v) + before * (np.abs(lat) @ np.abs(uv[h]).T)
                full = np.concatenate([k, kv[:, 512:]], axis=1)
                score = self.scale * (signed[b:e, h] @ full.T)
                f32 = 2.0 ** -16 * self.scale * (q[b:e, h] @ np.abs(full).T)
                d = self.scale * (q[b:e, h, :self.dn] @ k_off.T) + f32
                d[hidden], score[hidden] = 0.0, -np.inf
                top = d.max(axis=1, keepdims=True)
                peak = score.max(axis=1, keepdims=True)
                p = np.exp(score - np.where(np.isinf(peak), 0, peak))
                p /= np.maximum(p.sum(axis=1, keepdims=True), 1e-300)
                grow = (np.expm1(2 * top) + H) * (1 + H) + 2.0 ** -16
                off_out[b:e, h] = grow * (p @ np.abs(v)) + (1 + grow) * (p @ v_off)
                off_lse[b:e, h] = top[:, 0] + 2.0 ** -16 * (1 + np.abs(peak[:, 0]))
        return off_out, off_lse

    def check(self, covered=None, spread=True):
        torch.cuda.synchronize()
        ref, ref_lse = self.oracle()
        off_out, off_lse = self.bounds()
        got = f64(self.out)
        rows = slice(int(self.q_start[0]), int(self.q_start[-1]))
        ref, ref_lse, off_out, off_lse = ref[rows], ref_lse[rows], off_out[rows], off_lse[rows]
        nan = np.isnan(ref)
        np.testing.assert_array_equal(np.isnan(got[rows]), nan)
        half = H if self.out.dtype == torch.bfloat16 else 2.0 ** -24
        err = np.abs(got[rows] - ref)[~nan]
        allowed = (off_out + half * (np.abs(ref) + off_out))[~nan]
        assert (err <= allowed).all(), f"worst {float((err - allowed).max()):.3e}"
        norm = np.linalg.norm(ref[~nan])
        if spread and norm:
            assert np.linalg.norm(err) <= 1e-2 * norm, np.linalg.norm(err) / norm
        if self.lse is not None:
            lse = f64(self.lse)[rows]
            empty = np.isneginf(ref_lse)
            np.testing.assert_array_equal(np.isneginf(lse), empty)
            np.testing.assert_array_equal(np.isnan(lse), np.isnan(ref_lse))
            assert (got[rows][empty] == 0).all()
            live = np.isfinite(ref_lse)
            assert (np.abs(lse[live] - ref_lse[live]) <= off_lse[live]).all()
        for t, keep in ((self.out, 7.0), (self.lse, 7.0)):
            if t is not None:      # rows of no sequence
                assert (t[:rows.start] == keep).all() and (t[rows.stop:] == keep).all()


LENGTHS = [([1], [0]), ([1], [1]), ([5], [60]), ([64], [0]), ([128], [0]), ([129, 1], [0, 63]),
           ([256], [0]), ([257, 3], [127, 1000]), ([300], [517]), ([2, 1, 130, 63], [125, 128, 256, 0]),
           ([700], [0])]


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("new,cached", LENGTHS)
def test_lengths(cuda_device, fmt, new, cached):
    c = Case(cuda_device, fmt, new, cached, seed=sum(new))
    launch = c.launch()
    launch()
    assert launch.device_error() == 0
    c.check()


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("heads", [1, 16, 128])
def test_head_counts_and_f32_output(cuda_device, fmt, heads):
    c = Case(cuda_device, fmt, [37, 9], [101, 0], heads=heads)
    c.launch(out_dtype=torch.float32)()
    c.check()


@pytest.mark.parametrize("fmt", [1, 2])
def test_without_lse_and_rows_of_no_sequence_stay(cuda_device, fmt):
    c = Case(cuda_device, fmt, [3, 0, 140, 0], [70, 90, 0, 0], lead=4, tail=300)
    launch = c.launch(lse=False)
    launch()
    assert launch.device_error() == 0
    c.check()


def test_one_long_row_of_work(cuda_device):
    """Few query rows, many keys: the work of a unit is split and joined."""
    c = Case(cuda_device, 2, [40], [9001], heads=2, seed=4)
    c.launch()()
    c.check()


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("new,cached,heads", [([18, 353, 1], [3651, 0, 0], 3), ([2, 312], [4219, 403], 5),
                                              ([345, 6, 2, 75], [2130, 38, 101, 14], 2),
                                              ([1, 3, 280, 17, 4], [2231, 477, 3024, 0, 3], 2)])
def test_split_and_whole_blocks_together(cuda_device, fmt, new, cached, heads):
    """Blocks of very different lengths in one call: some are split over their keys, in different
    numbers of pieces, some are not."""
    c = Case(cuda_device, fmt, new, cached, heads=heads, seed=len(new))
    c.launch()()
    c.check()


def test_many_sequences(cuda_device):
    rng = np.random.default_rng(8)
    new, cached = rng.integers(0, 30, 1100), rng.integers(0, 3, 1100)
    c = Case(cuda_device, 2, new, cached, heads=1)
    c.launch()()
    c.check()


@pytest.mark.parametrize("fmt", [0, 2])
def test_positions_in_no_order_and_empty_rows(cuda_device, fmt):
    """A tree's or a reordered batch's positions: any row may see any prefix, or nothing."""
    c = Case(cuda_device, fmt, [150, 40], [200, 30], seed=6)
    rng = np.random.default_rng(1)
    c.q_pos = rng.integers(-3, 400, len(c.q_pos))
    c.q_pos[10:20] = -1
    c.q_pos[150:] = rng.integers(-2, 2 ** 31 - 1, 40)
    c.launch()()
    c.check()
    c.q_pos[:] = -1
    c.launch()()
    c.check()
    c.kv_len = np.array([0, -5])
    c.launch()()
    c.check()


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_strided_queries_outputs_weights_and_rows(cuda_device, fmt):
    c = Case(cuda_device, fmt, [70, 5], [61, 300], seed=2, row_pad=32)
    wide = torch.zeros((c.tokens, c.heads + 2, c.dn + c.dr + 8), dtype=torch.bfloat16, device=cuda_device)
    wide[:, 1:-1, :c.dn + c.dr] = c.q
    c.q = wide[:, 1:-1, :c.dn + c.dr]
    packed = torch.cat([c.w_uk, c.w_uv], dim=1).contiguous()
    c.w_uk, c.w_uv = packed[:, :c.dn], packed[:, c.dn:]
    c.launch()
    c.out = torch.full((c.tokens, c.heads + 1, c.dv + 16), 7.0, dtype=torch.bfloat16, device=cuda_device)
    whole, c.out = c.out, c.out[:, :c.heads, :c.dv]
    ops.MlaChunk(*c.args(), c.out, c.lse, scale=c.scale, kv_format=fmt, max_keys=c.max_keys + 1000)()
    c.check()
    assert (whole[:, c.heads:] == 7.0).all() and (whole[:, :, c.dv:] == 7.0).all()


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_a_row_that_is_not_finite_reaches_only_those_who_see_it(cuda_device, fmt):
    c = Case(cuda_device, fmt, [200, 30], [50, 100], seed=3)
    flat = c.kv.view(-1, c.kv.shape[-1])
    for position in (100, 230):       # of sequence 0
        row = int(c.table[0, position // 64]) * 64 + position % 64
        if fmt == 1:
            flat[row, 77] = 0x7F if position == 100 else 0xFF
        else:
            value = float("inf") if position == 100 else float("nan")
            at = 2 * (5 if position == 100 else (540 if fmt == 2 else 311))
            flat[row, at:at + 2] = torch.tensor([value], dtype=torch.bfloat16).view(torch.uint8).to(cuda_device)
    c.launch()()
    c.check()
    got = torch.isnan(c.out).all(dim=2).all(dim=1).cpu().numpy()
    np.testing.assert_array_equal(got, [50 + t >= 100 and t < 200 for t in range(230)])


@pytest.mark.parametrize("fmt", [0, 2])
def test_a_row_whose_expansion_overflows_reaches_only_those_who_see_it(cuda_device, fmt):
    """Finite latent values of 3e38: keys and values past bf16's range."""
    c = Case(cuda_device, fmt, [200], [50], seed=3)
    c.launch()()
    clean, clean_lse = c.out, c.lse
    row = int(c.table[0, 220 // 64]) * 64 + 220 % 64
    c.kv.view(-1, c.kv.shape[-1])[row, :1024] = torch.full((512,), 3e38, dtype=torch.bfloat16).view(torch.uint8).to(cuda_device)
    c.w_uv[0, 3] = c.w_uv[0, 3].abs()
    c.w_uk[1, 5] = c.w_uk[1, 5].abs()
    first = Case(cuda_device, fmt, [200], [50], seed=3)
    first.w_uv, first.w_uk = c.w_uv, c.w_uk
    first.launch()()
    c.launch()()
    seen = 170                       # tokens 0 to 169 are at positions below 220
    assert torch.equal(c.out[:seen], first.out[:seen]) and torch.equal(c.lse[:seen], first.lse[:seen])
    assert not torch.equal(clean[:seen], first.out[:seen])


@pytest.mark.parametrize("fmt", [0, 2])
def test_heads_in_several_passes(cuda_device, fmt):
    """A bound so large that the expanded keys and values of all heads do not fit the scratch."""
    c = Case(cuda_device, fmt, [140, 30], [200, 1500], heads=5, seed=8)
    launch = c.launch(max_keys=1 << 22)
    assert launch.workspace.numel() < 20 << 30
    launch()
    assert launch.device_error() == 0
    c.check()
    del launch
    torch.cuda.empty_cache()


def test_passes_without_a_join_between_them(cuda_device):
    """So many query blocks that none is split: the next pass's expansion directly follows an
    attention. The same sums in the same order as in one pass, so the same bits."""
    c = Case(cuda_device, 2, [1100, 500], [0, 300], heads=80, seed=22)
    c.launch()()
    torch.cuda.synchronize()
    want, want_lse = c.out, c.lse
    launch = c.launch(max_keys=280000)           # 59 heads a pass
    for _ in range(4):
        c.out.fill_(7.0)
        c.lse.fill_(7.0)
        launch()
        assert launch.device_error() == 0
        assert torch.equal(c.out, want) and torch.equal(c.lse, want_lse)
    sample = [0, 58, 59, 79]                     # heads of both passes against the oracle
    small = Case.__new__(Case)
    small.__dict__.update(c.__dict__)
    small.heads = len(sample)
    for name in ("q", "out", "lse"):
        setattr(small, name, getattr(c, name)[:, sample].contiguous())
    for name in ("w_uk", "w_uv"):
        setattr(small, name, getattr(c, name)[sample].contiguous())
    small.check()
    del launch
    torch.cuda.empty_cache()


@pytest.mark.parametrize("fmt", [0, 2])
def test_a_query_that_is_not_finite_stays_in_its_row(cuda_device, fmt):
    c = Case(cuda_device, fmt, [140], [20], seed=5)
    c.q[13, 1, 4] = float("nan")
    c.q[90, 2, 100] = float("inf")
    c.launch()()
    torch.cuda.synchronize()
    bad = torch.isnan(c.out).all(dim=2)
    assert bad[13, 1] and bad[90, 2] and int(bad.sum()) == 2 and int(torch.isnan(c.out).any(dim=2).sum()) == 2
    c.q[13, 1, 4] = c.q[90, 2, 100] = 0
    first = c.out
    c.launch()()
    keep = ~bad
    assert torch.equal(first[keep], c.out[keep])


@pytest.mark.parametrize("fmt", [0, 2])
@pytest.mark.parametrize("spread", [0.0, 12.0])
def test_flat_and_peaked_scores(cuda_device, fmt, spread):
    """Scores all equal, and scores spread over more than f32's exponent once exponentiated: the
    running maximum moves by large steps."""
    c = Case(cuda_device, fmt, [260], [300], heads=2, seed=7)
    c.q *= spread
    c.launch(out_dtype=torch.float32)()
    c.check(spread=spread == 0.0)


def test_scores_that_keep_growing(cuda_device):
    """Every row tile has a larger maximum than the one before: each one rescales the sums."""
    c = Case(cuda_device, 2, [130], [900], heads=2, seed=9)
    flat = c.kv.view(-1, 1152).view(torch.bfloat16)
    for position in range(1030):
        row = int(c.table[0, position // 64]) * 64 + position % 64
        flat[row, 512:576] = 0.0
        flat[row, 512] = position / 8.0
    c.q[:, :, 128] = 8.0
    c.launch(out_dtype=torch.float32)()
    c.check(spread=False)


def test_range_flags(cuda_device):
    c = Case(cuda_device, 2, [40, 8], [100, 100])
    c.table[0, 1] = 10 ** 6
    c.table[1, 0] = -1
    launch = c.launch()
    launch()
    assert launch.device_error() == _abi.DEV_PAGE_RANGE
    c.check()

    c = Case(cuda_device, 2, [40], [100])
    c.kv_len = np.array([10 ** 6])
    c.q_pos += 500
    launch = c.launch(max_keys=64 * c.table.shape[1])
    # the table's last page has stale rows behind the cached ones: give them values
    c.kv[int(c.table[0, -1])] = 0
    launch()
    assert launch.device_error() == _abi.DEV_TABLE_SHORT
    c.kv_len = np.array([64 * c.table.shape[1]])
    c.check()

    for bad in ([0, 30, 20], [0, 20, 49], [-1, 20, 48]):
        c = Case(cuda_device, 2, [40, 8], [100, 100])
        c.q_start = np.array(bad)
        launch = c.launch()
        launch()
        assert launch.device_error() == _abi.DEV_SEQ_RANGE
        assert (c.out == 7.0).all() and (c.lse == 7.0).all()

    c = Case(cuda_device, 2, [40, 8], [1000, 1000])
    launch = c.launch(max_keys=1000)
    launch()
    assert launch.device_error() == _abi.DEV_WORK_OVERFLOW
    assert (c.out == 7.0).all()


def test_refusals_raise(cuda_device):
    c = Case(cuda_device, 2, [4], [4])
    with pytest.raises(ops.ContractError) as e:
        c.launch(max_keys=1 << 30)
    assert (e.value.field, e.value.kind) == ("max_keys", 7)
    with pytest.raises(ops.TqError) as e:
        c.launch(workspace=torch.empty(64, dtype=torch.uint8, device=cuda_device))
    assert e.value.field == "workspace"
    with pytest.raises(ValueError, match="one CUDA device"):
        c.launch(workspace=torch.empty(1 << 30, dtype=torch.uint8))
    c.q = c.q[:, :, :128]
    with pytest.raises(ops.ContractError) as e:
        c.launch()
    assert (e.value.field, e.value.kind) == ("q", 1)


@pytest.mark.parametrize("fmt", [1, 2])
def test_replays_from_a_graph_with_other_contents(cuda_device, fmt):
    first = Case(cuda_device, fmt, [70, 200], [300, 11], seed=1, spare=20)
    launch = first.launch(max_keys=2000)
    launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        launch()
    graph.replay()
    first.check()
    once = first.out.clone()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(once, first.out)          # the same bits again
    # other lengths, positions and pages in the same buffers
    tensors = launch._keep
    first.q_start, first.kv_len = np.array([0, 255, 270]), np.array([290, 311])
    first.q_pos = np.concatenate([np.arange(35, 290), np.arange(296, 311)])
    tables = first.table.copy()
    first.table = np.full_like(tables, -1)
    pages = np.arange(first.kv.shape[0])[::-1]
    first.table[0, :5], first.table[1, :5] = pages[:5], pages[5:10]
    rng = np.random.default_rng(0)
    fill = Case(cuda_device, fmt, [1], [64 * first.kv.shape[0] - 1], seed=11, spare=0)
    first.kv.copy_(fill.kv)
    for at, value in ((4, first.table), (5, first.q_start), (6, first.q_pos), (7, first.kv_len)):
        tensors[at].copy_(i32(value, cuda_device))
    graph.replay()
    first.check()
    del graph, rng


def test_two_launches_on_two_streams(cuda_device):
    a, b = Case(cuda_device, 2, [200], [700], heads=8, seed=1), Case(cuda_device, 0, [300], [100], heads=4, seed=2)
    la, lb = a.launch(), b.launch()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        la(streams[0])
        lb(streams[1])
    torch.cuda.synchronize()
    a.check()
    b.check()


def test_a_call_on_another_stream_keeps_its_memory(cuda_device):
    """What a call allocates and drops on return is not handed to the current stream while the call
    still runs on its own."""
    c = Case(cuda_device, 2, [512], [1500], heads=16, seed=21)
    launch = c.launch()
    launch()
    torch.cuda.synchronize()
    need = launch.workspace.numel()
    want, want_lse = c.out.clone(), c.lse.clone()
    del launch
    side = torch.cuda.Stream()
    for _ in range(3):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        torch.zeros(need, dtype=torch.uint8, device=cuda_device)     # a free block of the current stream
        outs = []
        meta = [i32(x, cuda_device) for x in (c.table, c.q_start, c.q_pos, c.kv_len)]
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(3):
            outs.append(ops.mla_chunk(c.q, c.w_uk, c.w_uv, c.kv, *meta, scale=c.scale,
                                      max_keys=int(c.kv_len.sum()), stream=side))
            torch.full((need,), 255, dtype=torch.uint8, device=cuda_device)
        torch.cuda.synchronize()
        for out, lse in outs:
            assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_pages_past_four_gigabytes(cuda_device):
    c = Case(cuda_device, 2, [50], [200], seed=12)
    pages = 60000                                # 4.4 GB of 576-wide rows
    pool = torch.empty((pages, 64, 1152), dtype=torch.uint8, device=cuda_device)
    where = pages - 1 - 7 * np.arange(c.table.shape[1])
    ref = c.oracle()
    for i, p in enumerate(where):
        pool[int(p)] = c.kv[int(c.table[0, i])]
    small, c.kv, c.table = c.kv, pool, where[None].copy()
    c.launch()()
    torch.cuda.synchronize()
    c.kv, c.table = small, np.arange(len(where))[None]
    got = f64(c.out)
    assert np.linalg.norm(got - ref[0]) <= 1e-2 * np.linalg.norm(ref[0])
    del pool


def test_fp8_rows_match_their_bf16_operands(cuda_device):
    """FP8 rows and bf16 rows that hold their dequantized values give the same bits."""
    c = Case(cuda_device, 1, [100, 30], [77, 500], seed=4)
    c.launch()()
    rows = ofp8.operand_rows(c.kv.reshape(-1, 544).cpu().numpy())
    twin = Case(cuda_device, 1, [100, 30], [77, 500], seed=4)
    twin.fmt = 0
    twin.kv = bf16(np.nan_to_num(rows, nan=0.0), cuda_device).view(-1, 64, 512)
    twin.launch()()
    assert torch.equal(c.out, twin.out) and torch.equal(c.lse, twin.lse)
