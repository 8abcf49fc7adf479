"""Host validation of the chunk attention (tq_mla_chunk_validate, tq_mla_chunk_workspace_bytes) and
its oracle, CPU only: fake numeric addresses, the field names and violation kinds of the others."""

import ctypes

import numpy as np
import pytest

from oracle import chunk as ochunk
from oracle import mla as omla
from tq_mla import _abi

SHAPE, DTYPE, DIMENSION, STRIDE, ALIGNMENT, ADDRESS, CAPACITY, SCALE, ALIAS = 1, 2, 3, 4, 5, 6, 7, 10, 12
GiB = 1 << 30
PAYLOAD = {0: 1024, 1: 528, 2: 1152}


def tensor(shape, dtype, address):
    elem = {_abi.DTYPE_BF16: 2, _abi.DTYPE_U8: 1}.get(dtype, 4)
    t = _abi.TqTensorSpec()
    t.rank, t.dtype, t.device_address = len(shape), dtype, address
    stride = elem
    for i in reversed(range(len(shape))):
        t.shape[i], t.strides_bytes[i] = shape[i], stride
        stride *= shape[i]
    t.buffer_bytes = stride
    return t


def spec(tokens=9, heads=3, fmt=2, seqs=2, slots=4, pages=7, max_keys=500, out=None, lse=True):
    dn, dr = (128, 64) if fmt == 2 else (256, 0)
    bf, i32, f32 = _abi.DTYPE_BF16, _abi.DTYPE_I32, _abi.DTYPE_F32
    s = _abi.TqMlaChunkSpec()
    s.q = tensor([tokens, heads, dn + dr], bf, 1 * GiB)
    s.w_uk = tensor([heads, dn, 512], bf, 2 * GiB)
    s.w_uv = tensor([heads, dn, 512], bf, 3 * GiB)
    row = (PAYLOAD[fmt] + 15) // 16 * 16
    s.kv = tensor([pages, 64, row], _abi.DTYPE_U8, 4 * GiB)
    s.kv.shape[2] = PAYLOAD[fmt]
    s.page_table = tensor([seqs, slots], i32, 5 * GiB)
    s.q_start = tensor([seqs + 1], i32, 6 * GiB)
    s.q_pos = tensor([tokens], i32, 7 * GiB)
    s.kv_len = tensor([seqs], i32, 8 * GiB)
    s.out = tensor([tokens, heads, dn], bf if out is None else out, 9 * GiB)
    if lse:
        s.lse = tensor([tokens, heads], f32, 10 * GiB)
    s.kv_format, s.softmax_scale, s.max_keys = fmt, 0.1, max_keys
    return s


def verdict(s):
    err = _abi.TqContractError()
    st = _abi.lib.tq_mla_chunk_validate(ctypes.byref(s), ctypes.byref(err))
    return None if st == 0 else (err.field.decode(), st)


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_every_row_format_and_head_count_validates(fmt):
    for heads in (1, 3, 16, 128):
        assert verdict(spec(fmt=fmt, heads=heads)) is None
        assert verdict(spec(fmt=fmt, heads=heads, out=_abi.DTYPE_F32, lse=False)) is None
    assert verdict(spec(fmt=fmt, tokens=0)) is None
    assert verdict(spec(fmt=fmt, max_keys=0)) is None


def test_rejections_name_the_field_and_kind():
    assert verdict(spec(heads=129)) == ("q", SHAPE)
    s = spec(); s.kv_format = 7
    assert verdict(s) == ("kv_format", SHAPE)
    s = spec(); s.kv_format = 0
    assert verdict(s)[1] in (SHAPE, STRIDE)
    s = spec(); s.q.shape[2] = 576
    assert verdict(s) == ("q", SHAPE)
    for name in ("w_uk", "w_uv"):
        s = spec(); getattr(s, name).shape[1] = 64
        assert verdict(s) == (name, SHAPE)
        s = spec(); getattr(s, name).shape[0] = 2
        assert verdict(s) == (name, SHAPE)
    for name in ("q_start", "q_pos", "kv_len", "lse"):
        s = spec(); getattr(s, name).shape[0] += 1
        assert verdict(s) == (name, SHAPE), name
    for name in ("q", "w_uk", "w_uv", "out"):
        s = spec(); getattr(s, name).device_address += 8
        assert verdict(s) == (name, ALIGNMENT), name
        s = spec(); t = getattr(s, name); t.strides_bytes[0] += 8; t.buffer_bytes += 8 * t.shape[0]
        assert verdict(s) == (name, STRIDE), name
    for name in ("q", "w_uk", "w_uv", "kv", "page_table", "q_start", "q_pos", "kv_len", "out", "lse"):
        s = spec(); getattr(s, name).device_address = 0
        assert verdict(s) == (name, ADDRESS), name
        s = spec(); getattr(s, name).buffer_bytes = 4
        assert verdict(s) == (name, CAPACITY), name
        s = spec(); getattr(s, name).dtype = 9
        assert verdict(s) == (name, DTYPE), name
    s = spec(); s.kv.shape[0] = 1 << 25
    assert verdict(s) == ("kv", DIMENSION)
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        s = spec(); s.softmax_scale = bad
        assert verdict(s) == ("softmax_scale", SCALE)
    assert verdict(spec(max_keys=(1 << 24) + 1)) == ("max_keys", CAPACITY)


@pytest.mark.parametrize("out", ["out", "lse"])
@pytest.mark.parametrize("other", ["q", "w_uk", "w_uv", "kv", "page_table", "q_start", "q_pos", "kv_len"])
def test_outputs_never_overlap_an_input(out, other):
    s = spec()
    getattr(s, out).device_address = getattr(s, other).device_address
    assert verdict(s) == (out, ALIAS)


def test_slices_of_one_packed_weight_validate():
    s = spec()
    for name, at in (("w_uk", 0), ("w_uv", 128 * 1024)):
        t = getattr(s, name)
        t.device_address = 2 * GiB + at
        t.strides_bytes[0] = 256 * 1024
        t.buffer_bytes = 3 * 256 * 1024 - at
    assert verdict(s) is None


def test_workspace_grows_with_the_bound_and_refuses_bad_specs():
    n = ctypes.c_uint64()
    sizes = []
    for keys in (0, 1000, 100000):
        assert _abi.lib.tq_mla_chunk_workspace_bytes(ctypes.byref(spec(max_keys=keys)), 0, ctypes.byref(n)) == 0
        sizes.append(n.value)
    assert sizes[0] < sizes[1] < sizes[2] and sizes[1] > 1000 * 3 * 256 * 2
    # the scratch of one pass is bounded, whatever the number of heads
    big = spec(heads=128, max_keys=1 << 23)
    assert _abi.lib.tq_mla_chunk_workspace_bytes(ctypes.byref(big), 0, ctypes.byref(n)) == 0
    assert n.value < (8 << 30) + (1 << 23) * 1300 + (1 << 30)
    assert _abi.lib.tq_mla_chunk_workspace_bytes(ctypes.byref(spec(heads=129)), 0, ctypes.byref(n)) == SHAPE


@pytest.mark.parametrize("fmt", [0, 2])
def test_oracle_equals_the_absorbed_core(fmt):
    """Expanded keys and values against the absorbed core on the same rows (the RoPE part as 64
    more latent dimensions with an identity key weight and no value weight)."""
    rng = np.random.default_rng(3 + fmt)
    heads, slots, dr = 2, 3, 64 if fmt == 2 else 0
    dn = dv = 128 if fmt == 2 else 256
    rows = rng.standard_normal((8 * 64, 512 + dr))
    table = rng.permutation(8)[:6].reshape(2, slots)
    kv_len, q_start = np.array([150, 70]), np.array([0, 5, 12])
    q_pos = np.concatenate([np.arange(145, 150), np.arange(63, 70)])
    w_uk, w_uv = rng.standard_normal((2, heads, dn, 512)) / np.sqrt(512)
    q = rng.standard_normal((12, heads, dn + dr))
    out, lse = ochunk.chunk_attention(q, w_uk, w_uv, rows, table, q_start, q_pos, kv_len, scale=0.09, step=3)
    wide_uk = np.zeros((heads, dn + dr, 512 + dr))
    wide_uk[:, :dn, :512] = w_uk
    wide_uk[:, dn:, 512:] = np.eye(dr)
    wide_uv = np.concatenate([w_uv, np.zeros((heads, dv, dr))], axis=2)
    for s in range(2):
        b, e = q_start[s], q_start[s + 1]
        lat = omla.gather_rows(rows, table[s], kv_len[s])
        mask = np.arange(kv_len[s])[None] <= q_pos[b:e, None]
        ref, _, ref_lse = omla.mla_attention_core(q[b:e], lat, wide_uk, wide_uv, mask, scale=0.09)
        np.testing.assert_allclose(out[b:e], ref, rtol=1e-9, atol=1e-10)
        np.testing.assert_allclose(lse[b:e], ref_lse, rtol=1e-9)


def test_prologue_without_w_uk_declares_the_query_of_the_chunk():
    """A prologue whose w_uk has rank 0 takes q [T, H, Dn + Dr] and no space for a second one."""
    import test_prologue_contract as tp
    for dr, fmt in ((64, _abi.KV_BF16_ROPE576), (0, _abi.KV_FP8_E4M3)):
        s = tp.spec(dr=dr, fmt=fmt)
        n, m = ctypes.c_uint64(), ctypes.c_uint64()
        assert _abi.lib.tq_mla_prologue_workspace_bytes(ctypes.byref(s), ctypes.byref(n)) == 0
        s.w_uk = _abi.TqTensorSpec()
        assert tp.verdict(s) == ("q", SHAPE)
        s.q = tp.tensor([6, 4, 128 + dr], _abi.DTYPE_BF16, 12 * GiB, 2)
        assert tp.verdict(s) is None
        assert _abi.lib.tq_mla_prologue_workspace_bytes(ctypes.byref(s), ctypes.byref(m)) == 0
        assert m.value < n.value
        s.q.device_address = s.w_qb.device_address
        assert tp.verdict(s) == ("q", ALIAS)
