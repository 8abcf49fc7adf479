"""GPU: the device error flags after a call without tokens or without sequences are that call's, not
what the workspace held before."""

import pytest
import torch

from test_gpu_chunk import Case
from tq_mla import _abi, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("what", ["no tokens", "no sequences"])
def test_chunk_attention_of_nothing_clears_its_flags(cuda_device, fmt, what):
    c = Case(cuda_device, fmt, [4], [100])
    q, w_uk, w_uv, kv, table, q_start, q_pos, kv_len = c.args()
    if what == "no tokens":
        q, q_pos, q_start = q[:0], q_pos[:0], torch.zeros_like(q_start)
    else:
        table, q_start, kv_len = table[:0], q_start[:1], kv_len[:0]
    out = torch.full((q.shape[0], c.heads, c.dv), 7.0, dtype=torch.bfloat16, device=cuda_device)
    launch = ops.MlaChunk(q, w_uk, w_uv, kv, table, q_start, q_pos, kv_len, out, scale=c.scale, kv_format=fmt,
                          max_keys=200)
    launch.workspace.fill_(255)
    launch()
    assert launch.device_error() == 0
    assert (out == 7.0).all()


def test_flags_of_an_earlier_call_in_the_same_workspace_do_not_stay(cuda_device):
    c = Case(cuda_device, 2, [40, 8], [100, 100])
    c.table[0, 1] = 10 ** 6
    launch = c.launch()
    launch()
    assert launch.device_error() == _abi.DEV_PAGE_RANGE
    q, w_uk, w_uv, kv, table, q_start, q_pos, kv_len = c.args()
    empty = ops.MlaChunk(q[:0], w_uk, w_uv, kv, table, q_start * 0, q_pos[:0], kv_len, c.out[:0], scale=c.scale,
                         kv_format=2, max_keys=200, workspace=launch.workspace)
    empty()
    assert empty.device_error() == 0


def test_attention_of_no_tokens_reports_no_flags(cuda_device):
    b = torch.zeros((2, 64, 1152), dtype=torch.uint8, device=cuda_device)
    i = torch.zeros((1, 2), dtype=torch.int32, device=cuda_device)
    q = torch.zeros((0, 16, 576), dtype=torch.bfloat16, device=cuda_device)
    for prefill in (False, True):
        launch = ops.MlaLaunch(q, b, i, i[0, :0], i[0, :0], i[0, :1], q[:, :, :512].contiguous(),
                               torch.zeros((0, 16), device=cuda_device), scale=0.1, query_counts=[0],
                               prefill=prefill)
        launch.workspace.fill_(255)
        launch()
        assert launch.device_error() == 0
