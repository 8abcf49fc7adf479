"""GPU: a one-shot chunk attention reports what it left out (``flags``), and the results that it
allocates hold NaN in the rows that it did not compute, never what the memory held before."""

import numpy as np
import pytest
import torch

from test_gpu_chunk import Case, i32
from tq_mla import _abi, ops

pytestmark = pytest.mark.gpu


def one_shot(c, flags=None, **kw):
    kw.setdefault("max_keys", c.max_keys)
    # what the allocator hands out next holds ordinary numbers
    for n in (c.tokens * c.heads * c.dv * 2, c.tokens * c.heads * 4):
        torch.zeros(n, dtype=torch.uint8, device=c.device)
    return ops.mla_chunk(*c.args(), scale=c.scale, kv_format=c.fmt, flags=flags, **kw)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("what", ["bound", "order"])
def test_a_call_that_is_left_out_says_so(cuda_device, what, out_dtype):
    c = Case(cuda_device, 2, [40, 8], [1000, 1000])
    flags = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    if what == "order":
        c.q_start = np.array([0, 30, 20])
        out, lse = one_shot(c, flags, out_dtype=out_dtype)
        assert int(flags) == _abi.DEV_SEQ_RANGE
    else:
        out, lse = one_shot(c, flags, out_dtype=out_dtype, max_keys=1000)
        assert int(flags) == _abi.DEV_WORK_OVERFLOW
    assert out.dtype == out_dtype and torch.isnan(out).all() and torch.isnan(lse).all()


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_flags_of_a_call_that_is_computed(cuda_device, fmt):
    c = Case(cuda_device, fmt, [40, 8], [100, 100], lead=3, tail=5)
    flags = torch.full((2,), 64, dtype=torch.int32, device=cuda_device)
    out, lse = one_shot(c, flags)
    assert flags.tolist() == [64, 64]                           # bits are added, none are cleared
    c.launch()()
    rows = slice(3, 51)
    assert torch.equal(out[rows], c.out[rows]) and torch.equal(lse[rows], c.lse[rows])
    for t in (out, lse):                                        # rows of no sequence
        assert torch.isnan(t[:3]).all() and torch.isnan(t[51:]).all()
    c.table[0, 1] = 10 ** 6
    got = one_shot(c, flags)
    assert flags.tolist() == [64 | _abi.DEV_PAGE_RANGE, 64]
    assert torch.isfinite(got[0][rows].float()).all()
    mine = torch.full_like(c.out, 7.0), torch.full_like(c.lse, 7.0)
    one_shot(c, out=mine[0], lse=mine[1])                       # the caller's own rows stay as they were
    assert (mine[0][:3] == 7.0).all() and (mine[1][51:] == 7.0).all()


def test_flags_on_another_stream_and_without_tokens(cuda_device):
    c = Case(cuda_device, 2, [40, 8], [1000, 1000])
    flags = torch.zeros((), dtype=torch.int32, device=cuda_device)
    side = torch.cuda.Stream()
    meta = [i32(x, cuda_device) for x in (c.table, c.q_start, c.q_pos, c.kv_len)]
    torch.cuda.synchronize()
    out, _ = ops.mla_chunk(c.q, c.w_uk, c.w_uv, c.kv, *meta, scale=c.scale, max_keys=1000, flags=flags, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert int(flags) == _abi.DEV_WORK_OVERFLOW and torch.isnan(out).all()
    flags.zero_()
    out, lse = ops.mla_chunk(c.q[:0], c.w_uk, c.w_uv, c.kv, meta[0], meta[1] * 0, meta[2][:0], meta[3], scale=c.scale,
                             max_keys=1000, flags=flags)
    assert int(flags) == 0 and out.shape == (0, c.heads, c.dv) and lse.shape == (0, c.heads)
