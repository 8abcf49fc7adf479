"""GPU: the index key's norm where its factor and its weight are large and the values small."""

import numpy as np
import pytest
import torch

from oracle import index as oindex
from test_gpu_index import DIM, PAGE, ROW, bf16, check_rows, host, i32
from tq_mla import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bias", [False, True])
def test_small_keys_and_large_weights(cuda_device, bias):
    """A row of zeros is normalised to zeros (plus the bias) and a row far below the root of eps to its value
    times weight / sqrt(eps), although weight / sqrt(eps) alone is past the largest f32."""
    rng = np.random.default_rng(bias)
    eps = 1e-12
    k = np.zeros((4, DIM))
    k[1] = rng.standard_normal(DIM) * 2.0 ** -50
    k[2, ::2], k[2, 1::2] = 2.0 ** -60, -(2.0 ** -60)
    k[3] = rng.standard_normal(DIM)
    k = bf16(k, cuda_device)
    weight = bf16(2.0 ** 112 * (1 + rng.random(DIM)), cuda_device)
    assert (host(weight) / np.sqrt(eps) > np.finfo(np.float32).max).all()
    shift = bf16(2.0 ** 60 * rng.standard_normal(DIM), cuda_device) if bias else None
    kv = torch.full((1, PAGE, ROW), 9, dtype=torch.uint8, device=cuda_device)
    ops.index_write(None, k, None, i32([[0]], cuda_device), i32([0] * 4, cuda_device), i32(range(4), cuda_device), kv,
                    norm_weight=weight, norm_bias=shift, eps=eps)
    got = kv[0, :4].cpu().numpy()
    scale = np.ascontiguousarray(got[:, 128:132]).view(np.float32)[:, 0].astype(np.float64)
    want = oindex.normalised(host(k), host(weight), None if shift is None else host(shift), eps)
    assert np.isfinite(scale).all()
    if not bias:
        assert (got[0, :132] == 0).all() and not want[0].any()
        check_rows(got[1:, :DIM], scale[1:], want[1:])
    else:
        check_rows(got[:, :DIM], scale, want)
