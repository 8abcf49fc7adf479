"""Calls of the index branch that are refused because of a size or an argument that its kernels cannot take as
it is. CPU only."""

import pytest
import torch

from test_index_contract import DIMENSION, GiB, OK, SHAPE, STRIDE, changed, verdict, write
from tq_mla import ops

OVERFLOW = 8


def test_heads_too_far_apart():
    far = 1 << 36
    spread = lambda stride, heads=2: changed(  # noqa: E731
        write(tokens=1, heads=heads), "q", strides_bytes=[heads * stride, stride, 2], device_address=1000 * GiB,
        buffer_bytes=heads * stride)
    assert verdict(spread(far - 16)) == OK
    assert verdict(spread(far)) == ("q", OVERFLOW)
    assert verdict(spread(3 * far)) == ("q", OVERFLOW)
    assert verdict(spread(far, heads=1)) == OK           # nothing is a head's distance away


def test_pools_whose_rows_are_not_132_bytes_in_a_row():
    """What the kernels would write beside the tensor that they are given."""
    whole = torch.zeros((3, 64, 288), dtype=torch.uint8)
    for kv, kind in ((whole[..., ::2], STRIDE), (whole[..., :131], SHAPE), (whole[..., :128], SHAPE), (whole[0], SHAPE),
                     (torch.zeros((3, 64, 32), dtype=torch.float32), SHAPE)):
        with pytest.raises(ops.ContractError) as e:
            ops.index_pool_spec(kv)
        assert (e.value.field, e.value.kind) == ("kv", kind)
    for kv in (whole, whole[..., :132], whole[..., 16:], torch.zeros((3, 64, 36), dtype=torch.float32)):
        s = ops.index_pool_spec(kv)
        assert list(s.shape) == [3, 64, 132] and s.strides_bytes[2] == 1
        assert s.strides_bytes[1] == kv.stride(1) * kv.element_size()


@pytest.mark.parametrize("field", ["keep_first", "keep_last", "rope_start"])
@pytest.mark.parametrize("value", [2 ** 32, 2 ** 32 + 8, 2 ** 31, -2 ** 32, -2 ** 31 - 1])
def test_numbers_past_32_bits(field, value):
    """Their low 32 bits would be numbers that are accepted."""
    i, f = torch.zeros(1, dtype=torch.int32), torch.zeros((1, 9))
    with pytest.raises(ops.ContractError) as e:
        if field == "rope_start":
            kv = torch.zeros((1, 64, 144), dtype=torch.uint8)
            ops.index_write_spec(None, torch.zeros((1, 128), dtype=torch.bfloat16), None, i[None], i, i, kv, None, None, rope_start=value)
        else:
            ops.index_select_spec(f, i, i, i, i[None], i, **{field: value})
    assert (e.value.field, e.value.kind) == (field, DIMENSION)
