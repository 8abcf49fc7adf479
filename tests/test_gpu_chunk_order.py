"""GPU: chunk attention where a row's reference maximum moves in every tile, in all row formats.

The scores' growth comes from one component of the latent row that every rounding point keeps exactly
(multiples of 16 up to 240, with a key weight of one and nothing beside it), so what the roundings move
is the rest of the score, of unit spread, and the tolerances are those of test_gpu_chunk.py: its bound
of each element, and 1e-2 of the relative 2-norm."""

import numpy as np
import pytest
import torch

from test_gpu_chunk import Case, bf16

pytestmark = pytest.mark.gpu


def growing(device, fmt, new, cached, level, heads, seed):
    """A batch whose cached row n carries ``level(n)`` (exact in bf16) in a component that adds
    ``scale * 8 * level(n)`` to every score."""
    c = Case(device, fmt, new, cached, heads=heads, seed=seed)
    flat = c.kv.view(-1, c.kv.shape[-1])
    for s, n in enumerate(c.kv_len):
        pos = np.arange(n)
        rows = torch.from_numpy(c.table[s, pos // 64].astype(np.int64) * 64 + pos % 64).to(device)
        value = np.array([level(p) for p in pos], dtype=np.float32)
        if fmt == 1:
            # the whole tile of 128 values is that component: code 1.0 times the scale
            flat[rows, :128] = 0
            flat[rows, 0] = 0x38
            scale = torch.from_numpy(value).view(torch.uint8).view(-1, 4).to(device)
            flat[rows, 512:516] = scale
        else:
            flat[rows, :2] = bf16(value, device).view(torch.uint8).view(-1, 2)
    # component 0 of the key is component 0 of the latent row, and of nothing else
    c.w_uk[:, :, 0] = 0
    c.w_uk[:, 0] = 0
    c.w_uk[:, 0, 0] = 1
    c.w_uv[:, :, 0] = 0
    c.q[:, :, 0] = 8
    return c


# At 256 columns a step of 16 a tile is scale * 8 * 16 = 8 nats, 11.5 in log2 units (the reference
# moves by more than 8); at 192 columns 13.3.
LEVELS = {
    "every tile": lambda n: 16.0 * min(n // 128, 15),
    "every other tile": lambda n: 16.0 * min(n // 256, 15),
    "one key of a tile": lambda n: 16.0 * min(n // 128, 15) if n % 128 == 77 else 0.0,
    "falling": lambda n: max(0.0, 128.0 - 16.0 * (n // 128)),
}


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("name", sorted(LEVELS))
@pytest.mark.parametrize("new,cached,heads", [([130], [900], 2), ([300, 5, 513], [700, 1200, 0], 5)])
def test_a_reference_that_moves_in_every_tile(cuda_device, fmt, name, new, cached, heads):
    c = growing(cuda_device, fmt, new, cached, LEVELS[name], heads, seed=31)
    launch = c.launch(out_dtype=torch.float32)
    launch()
    assert launch.device_error() == 0
    c.check()
    want, want_lse = c.out.clone(), c.lse.clone()
    for _ in range(20):
        c.out.fill_(7.0)
        launch()
        assert torch.equal(c.out, want) and torch.equal(c.lse, want_lse)


@pytest.mark.parametrize("fmt", [0, 1])
def test_many_units_with_a_moving_reference(cuda_device, fmt):
    """All CTA pairs at work, several units each, so that the softmax groups drift apart: the same
    bits in every call, and the oracle's values for a sample of the heads."""
    c = growing(cuda_device, fmt, [1500, 700], [300, 1300], LEVELS["every tile"], 64, seed=33)
    launch = c.launch()
    launch()
    assert launch.device_error() == 0
    want, want_lse = c.out.clone(), c.lse.clone()
    for _ in range(30):
        launch()
        assert torch.equal(c.out, want) and torch.equal(c.lse, want_lse)
    sample = [0, 31, 63]
    small = Case.__new__(Case)
    small.__dict__.update(c.__dict__)
    small.heads = len(sample)
    for tensor in ("q", "out", "lse"):
        setattr(small, tensor, getattr(c, tensor)[:, sample].contiguous())
    for tensor in ("w_uk", "w_uv"):
        setattr(small, tensor, getattr(c, tensor)[sample].contiguous())
    small.check()
