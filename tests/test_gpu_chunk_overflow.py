"""GPU: finite cached rows whose expanded keys and values pass f32's range with both signs. A token
that does not see such a row gives the same bits as without it: the expansion of finite rows with
finite weights is never NaN (an infinite value in a tile would meet hidden weights of zero, so it is
cut to bf16's largest; a NaN could not be)."""

import numpy as np
import pytest
import torch

from test_gpu_chunk import Case

pytestmark = pytest.mark.gpu
POSITION = 220
SEEN_FROM = POSITION - 50      # the first token that sees it: 50 cached rows


def write_row(c, values):
    """512 latent values of magnitude about 3e38 at POSITION of sequence 0."""
    row = int(c.table[0, POSITION // 64]) * 64 + POSITION % 64
    flat = c.kv.view(-1, c.kv.shape[-1])
    if c.fmt == 1:
        flat[row, :512] = torch.where(values < 0, 0xFE, 0x7E).to(torch.uint8).to(c.device)   # -+448
        flat[row, 512:528] = torch.full((4,), 3e38 / 448).view(torch.uint8).to(c.device)
    else:
        flat[row, :1024] = values.to(torch.bfloat16).view(torch.uint8).to(c.device)


def signs(kind):
    i = torch.arange(512)
    return {"same": torch.ones(512), "alternating": 1.0 - 2.0 * (i % 2), "by steps": 1.0 - 2.0 * ((i // 16) % 2),
            "by halves": 1.0 - 2.0 * (i // 256)}[kind]


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("kind", ["same", "alternating", "by steps", "by halves"])
@pytest.mark.parametrize("spread", [0.15, 1.0, 1e30])
def test_hidden_rows_that_overflow_with_both_signs(cuda_device, fmt, kind, spread):
    c = Case(cuda_device, fmt, [200], [50], heads=4, seed=3)
    rng = np.random.default_rng(7)
    w = rng.standard_normal((4, c.dv, 512)) * spread
    w[3] = np.abs(w[3])            # one head whose partial sums follow the row's own signs
    if spread > 1e3:               # such weights overflow with the row alone: the others hold zeros
        flat = c.kv.view(-1, c.kv.shape[-1])
        flat[torch.from_numpy(c.live).to(cuda_device), :1024 if fmt != 1 else 512] = 0
    c.w_uv = torch.from_numpy(w).to(torch.bfloat16).to(cuda_device)
    if spread == 1.0:
        c.w_uk = c.w_uv.clone()
    c.launch()()
    torch.cuda.synchronize()
    want, want_lse = c.out[:SEEN_FROM].clone(), c.lse[:SEEN_FROM].clone()
    assert torch.isfinite(want).all() and torch.isfinite(want_lse).all()
    write_row(c, 3e38 * signs(kind))
    c.launch()()
    torch.cuda.synchronize()
    assert torch.equal(c.out[:SEEN_FROM], want) and torch.equal(c.lse[:SEEN_FROM], want_lse)
    # those that see it are not left at ordinary values
    assert not torch.isfinite(c.out[SEEN_FROM:].float()).all() or (c.out[SEEN_FROM:].float().abs() > 1e30).any()
