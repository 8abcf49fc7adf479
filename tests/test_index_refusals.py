"""Calls of the index branch that are refused because of a size or an argument that its kernels cannot take as
it is. CPU only."""

from test_index_contract import GiB, OK, changed, verdict, write

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
