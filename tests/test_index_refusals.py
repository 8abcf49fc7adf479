"""Calls of the index branch that are refused because of a size or an argument that its kernels cannot take as
it is. CPU only."""

import pytest
import torch

from test_index_contract import GiB, OK, SHAPE, STRIDE, changed, verdict, write
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
