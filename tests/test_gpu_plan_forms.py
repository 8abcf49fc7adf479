"""GPU: forms of the step plan's declaration that the bound object does not make (no slot, outputs at
any 4-byte address), a chunk attention whose sequences have no tokens, and flags that are refused."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import step as ostep
from test_gpu_chunk import Case
from test_gpu_step import _i32, _step
from tq_mla import _abi, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests,tokens", [(50, 401), (3000, 20003), (4500, 30001), (50, (1 << 19) + 3)])
@pytest.mark.parametrize("slot", [True, False])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_outputs_at_any_address_and_without_slots(cuda_device, requests, tokens, slot, shift):
    rng = np.random.default_rng(requests + shift)
    cached, new = rng.integers(0, 200, requests), rng.integers(0, 7, requests)
    table, free = _step(rng, requests, cached, new, 5)
    want = ostep.step_plan(cached, new, table, free, len(free), tokens)

    def out(n):     # n values with four more on each side, `shift` values off a 16-byte border
        whole = torch.full((n + 12,), 77, dtype=torch.int32, device=cuda_device)
        return whole, whole[4 + shift:4 + shift + n]

    places = {k: out(n) for k, n in dict(q_start=requests + 1, kv_len=requests, seq_id=tokens, q_pos=tokens,
                                         slot=tokens, free_left=1).items()}
    inputs = [_i32(a, cuda_device) for a in (cached, new, table, free, [len(free)])]
    d_table = inputs[2]
    outputs = [places[k][1] for k in ("q_start", "kv_len", "seq_id", "q_pos")]
    spec = ops.step_plan_spec(*inputs, *outputs, places["slot"][1] if slot else None, places["free_left"][1])
    flags = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    err = _abi.TqContractError()
    stream = torch.cuda.current_stream().cuda_stream
    assert _abi.lib.tq_step_plan(ctypes.byref(spec), flags.data_ptr(), stream, ctypes.byref(err)) == 0
    torch.cuda.synchronize()
    for name, ref in zip(("q_start", "kv_len", "seq_id", "q_pos", "slot"), want):
        whole, part = places[name]
        if name == "slot" and not slot:
            assert (whole == 77).all()
            continue
        np.testing.assert_array_equal(part.cpu().numpy(), ref, err_msg=name)
        assert (whole[:4 + shift] == 77).all() and (whole[4 + shift + len(part):] == 77).all()
    np.testing.assert_array_equal(d_table.cpu().numpy(), want[5])
    assert int(places["free_left"][1]) == want[6] and int(flags) == want[7]


def test_flags_have_to_be_int32_on_the_tensors_device(cuda_device):
    i = _i32([3], cuda_device)
    table = _i32([[0, 1]], cuda_device)
    plan = ops.StepPlan(i, i, table, _i32([4, 5], cuda_device), _i32([2], cuda_device), tokens=3)
    for bad in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64, device=cuda_device),
                torch.zeros(0, dtype=torch.int32, device=cuda_device)):
        with pytest.raises(ValueError, match="flags"):
            plan(bad)
    c, i32_table = Case(cuda_device, 2, [4], [9]), _i32([[0]], cuda_device)
    for bad in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64, device=cuda_device)):
        with pytest.raises(ValueError, match="flags"):
            ops.mla_chunk(*c.args(), scale=c.scale, max_keys=c.max_keys, flags=bad)
        with pytest.raises(ValueError, match="flags"):
            ops.kv_write(torch.zeros((1, 576), dtype=torch.bfloat16, device=cuda_device), c.kv, i32_table, i, i,
                         flags=bad)


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_chunk_attention_with_rows_of_no_sequence_alone(cuda_device, fmt):
    c = Case(cuda_device, fmt, [40, 8], [100, 100])
    for start in ([0, 0, 0], [48, 48, 48], [13, 13, 13]):
        c.q_start = np.array(start)
        launch = c.launch()
        launch()
        assert launch.device_error() == 0
        assert (c.out == 7.0).all() and (c.lse == 7.0).all()
