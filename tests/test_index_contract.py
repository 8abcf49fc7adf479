"""Host validation of the index branch (tq_index_write_validate, tq_index_scores_validate,
tq_index_select_validate), CPU only: fake numeric addresses, the field names and violation kinds of
the other contracts; struct layouts; the frequency table."""

import ctypes
import math
import subprocess

import pytest
import torch

from conftest import ROOT

from tq_mla import _abi, ops

SHAPE, DTYPE, DIMENSION, STRIDE, ALIGNMENT, ADDRESS, CAPACITY, SCALE, ALIAS = 1, 2, 3, 4, 5, 6, 7, 10, 12
GiB = 1 << 30
BF, I32, F32, U8 = _abi.DTYPE_BF16, _abi.DTYPE_I32, _abi.DTYPE_F32, _abi.DTYPE_U8
SIZE = {BF: 2, I32: 4, F32: 4, U8: 1}


def tensor(shape, dtype, place, strides=None):
    t = _abi.TqTensorSpec()
    t.rank, t.dtype, t.device_address = len(shape), dtype, place * GiB
    if strides is None:
        strides = [SIZE[dtype]]
        for d in reversed(shape[1:]):
            strides.append(strides[-1] * max(d, 1))
        strides.reverse()
    for i, (d, s) in enumerate(zip(shape, strides)):
        t.shape[i], t.strides_bytes[i] = d, s
    t.buffer_bytes = max(shape[0], 1) * strides[0]
    return t


def pool(place, pages=9, row=144):
    return tensor([pages, 64, 132], U8, place, [64 * row, row, 1])


def write(tokens=6, heads=16, queries=True, w_type=BF, norm=2, rope=32, start=0):
    s = _abi.TqIndexWriteSpec()
    if queries:
        s.q = tensor([tokens, heads, 128], BF, 1)
        s.w = tensor([tokens, heads], w_type, 2)
        s.q_out = tensor([tokens, heads, 128], U8, 3)
        s.w_out = tensor([tokens, heads], F32, 4)
    s.k = tensor([tokens, 128], BF, 5)
    s.page_table = tensor([3, 7], I32, 6)
    s.seq_id, s.pos = tensor([tokens], I32, 7), tensor([tokens], I32, 8)
    s.kv = pool(9)
    if norm:
        s.norm_weight = tensor([128], BF, 10)
    if norm > 1:
        s.norm_bias = tensor([128], BF, 11)
    if rope:
        s.freq = tensor([rope // 2], F32, 12)
    s.rope_start, s.rope_half, s.rope_mscale, s.norm_eps, s.scale = start, 0, 1.0, 1e-6, 0.1
    return s


def scores(tokens=6, heads=16, columns=500):
    s = _abi.TqIndexScoresSpec()
    s.q, s.w = tensor([tokens, heads, 128], U8, 1), tensor([tokens, heads], F32, 2)
    s.kv, s.page_table = pool(3), tensor([3, 7], I32, 4)
    s.seq_id, s.q_pos, s.kv_len = tensor([tokens], I32, 5), tensor([tokens], I32, 6), tensor([3], I32, 7)
    s.scores = tensor([tokens, columns], F32, 8)
    return s


def select(tokens=6, columns=500, k=20, pages=False, first=0, last=0):
    s = _abi.TqIndexSelectSpec()
    s.scores = tensor([tokens, columns], F32, 1)
    s.seq_id, s.q_pos, s.kv_len = tensor([tokens], I32, 2), tensor([tokens], I32, 3), tensor([3], I32, 4)
    if pages:
        s.page_table = tensor([3, 7], I32, 5)
    s.idx, s.len = tensor([tokens, k], I32, 6), tensor([tokens], I32, 7)
    s.keep_first, s.keep_last = first, last
    return s


def verdict(s):
    name = {_abi.TqIndexWriteSpec: "write", _abi.TqIndexScoresSpec: "scores",
            _abi.TqIndexSelectSpec: "select"}[type(s)]
    err = _abi.TqContractError()
    st = getattr(_abi.lib, f"tq_index_{name}_validate")(ctypes.byref(s), ctypes.byref(err))
    assert st == err.kind
    return (err.field.decode() if err.field else None, st)


OK = (None, 0)


@pytest.mark.parametrize("s", [
    write(), write(heads=1), write(heads=128), write(queries=False), write(w_type=F32), write(norm=0),
    write(norm=1), write(rope=0), write(rope=128), write(rope=16, start=112), write(tokens=0),
    scores(), scores(heads=8), scores(heads=128), scores(tokens=0), scores(columns=0),
    select(), select(k=2051), select(k=1), select(pages=True), select(first=7, last=13), select(tokens=0),
    select(columns=0), select(columns=1 << 20)])
def test_accepted(s):
    assert verdict(s) == OK


def changed(s, name, **fields):
    t = getattr(s, name)
    for key, value in fields.items():
        if key in ("shape", "strides_bytes"):
            for i, v in enumerate(value):
                getattr(t, key)[i] = v
        else:
            setattr(t, key, value)
    return s


def with_(s, **fields):
    for name, value in fields.items():
        setattr(s, name, value)
    return s


@pytest.mark.parametrize("s,want", [
    # write
    (write(heads=129), ("q", SHAPE)),
    (write(heads=0), ("q", SHAPE)),
    (changed(write(), "k", rank=1), ("k", SHAPE)),
    (changed(write(), "k", shape=[6, 64]), ("k", SHAPE)),
    (changed(write(), "k", strides_bytes=[264, 2], buffer_bytes=4096), ("k", STRIDE)),
    (changed(write(), "k", strides_bytes=[272, 2]), ("k", CAPACITY)),
    (changed(write(), "q", device_address=GiB + 8), ("q", ALIGNMENT)),
    (changed(write(), "q_out", device_address=3 * GiB + 8), ("q_out", ALIGNMENT)),
    (changed(write(), "q_out", rank=0), ("q_out", SHAPE)),
    (changed(write(), "w_out", rank=0), ("w_out", SHAPE)),
    (changed(write(), "w", rank=0), ("w", SHAPE)),
    (changed(write(), "w", dtype=I32), ("w", DTYPE)),
    (changed(write(), "w", device_address=0), ("w", ADDRESS)),
    (changed(write(), "norm_weight", rank=0), ("norm_weight", SHAPE)),
    (changed(write(), "norm_bias", shape=[64]), ("norm_bias", SHAPE)),
    (with_(write(), norm_eps=0.0), ("norm_eps", SCALE)),
    (with_(write(), norm_eps=math.nan), ("norm_eps", SCALE)),
    (with_(write(), scale=math.inf), ("scale", SCALE)),
    (with_(write(), rope_mscale=math.nan), ("rope_mscale", SCALE)),
    (write(rope=24), ("freq", SHAPE)),
    (write(rope=144), ("freq", SHAPE)),
    (write(rope=32, start=100), ("rope_start", SHAPE)),
    (write(rope=32, start=104), ("rope_start", SHAPE)),
    (write(rope=32, start=-8), ("rope_start", SHAPE)),
    (with_(write(), kv=pool(9, row=132)), ("kv", STRIDE)),
    (with_(write(), kv=pool(9, row=136)), ("kv", STRIDE)),
    (changed(write(), "kv", buffer_bytes=9 * 64 * 144 - 13), ("kv", CAPACITY)),
    (changed(write(), "kv", device_address=GiB), ("kv", ALIAS)),
    (changed(write(), "w_out", device_address=3 * GiB + 64), ("w_out", ALIAS)),
    (changed(write(), "seq_id", shape=[5]), ("seq_id", SHAPE)),
    # scores
    (scores(heads=4), ("q", SHAPE)),
    (scores(heads=12), ("q", SHAPE)),
    (scores(heads=136), ("q", SHAPE)),
    (changed(scores(), "q", dtype=BF), ("q", DTYPE)),
    (changed(scores(), "q", strides_bytes=[4096, 128, 1]), ("q", STRIDE)),
    (changed(scores(), "q", device_address=GiB + 4), ("q", ALIGNMENT)),
    (changed(scores(), "w", device_address=2 * GiB + 4), ("w", ALIGNMENT)),
    (changed(scores(), "w", shape=[6, 8]), ("w", SHAPE)),
    (changed(scores(), "kv_len", shape=[4]), ("kv_len", SHAPE)),
    (changed(scores(), "scores", shape=[5, 500]), ("scores", SHAPE)),
    (changed(scores(), "scores", dtype=BF), ("scores", DTYPE)),
    (changed(scores(), "scores", strides_bytes=[1600, 4]), ("scores", STRIDE)),
    (changed(scores(), "scores", device_address=2 * GiB), ("scores", ALIAS)),
    (changed(scores(), "kv", shape=[1 << 25, 64, 132]), ("kv", DIMENSION)),
    (with_(scores(), kv=pool(3, row=128)), ("kv", STRIDE)),
    # select
    (select(k=0), ("idx", SHAPE)),
    (select(k=2052), ("idx", SHAPE)),
    (select(columns=(1 << 20) + 1), ("scores", SHAPE)),
    (select(first=21), ("keep_first", SHAPE)),
    (select(first=-1), ("keep_first", SHAPE)),
    (select(first=10, last=11), ("keep_last", SHAPE)),
    (select(last=-1), ("keep_last", SHAPE)),
    (changed(select(), "idx", shape=[5, 20]), ("idx", SHAPE)),
    (changed(select(), "idx", strides_bytes=[96, 4]), ("idx", STRIDE)),
    (changed(select(), "len", dtype=F32), ("len", DTYPE)),
    (changed(select(pages=True), "page_table", shape=[4, 7]), ("page_table", SHAPE)),
    (changed(select(pages=True), "page_table", rank=1), ("page_table", SHAPE)),
    (changed(select(), "len", device_address=6 * GiB), ("len", ALIAS)),
])
def test_refused(s, want):
    assert verdict(s) == want


def test_null_specs_are_refused():
    for name in ("write", "scores", "select"):
        err = _abi.TqContractError()
        assert getattr(_abi.lib, f"tq_index_{name}_validate")(None, ctypes.byref(err)) == 100
        assert getattr(_abi.lib, f"tq_index_{name}")(None, None, None, ctypes.byref(err)) == 100


def test_refused_before_anything_is_launched():
    err = _abi.TqContractError()
    s = scores(heads=12)
    assert _abi.lib.tq_index_scores(ctypes.byref(s), None, None, ctypes.byref(err)) == SHAPE
    assert err.field == b"q"


def test_calls_without_tokens_need_no_device():
    for s, fn in ((write(tokens=0), "write"), (scores(tokens=0), "scores"), (select(tokens=0), "select")):
        err = _abi.TqContractError()
        assert getattr(_abi.lib, f"tq_index_{fn}")(ctypes.byref(s), None, None, ctypes.byref(err)) == 0


def test_struct_layouts(tmp_path):
    header = ROOT / "include" / "tq_mla.h"
    structs = (_abi.TqIndexWriteSpec, _abi.TqIndexScoresSpec, _abi.TqIndexSelectSpec)
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(){"]
    for c in structs:
        lines.append(f'printf("{c.__name__} %zu\\n", sizeof({c.__name__}));')
        lines += [f'printf("{c.__name__}.{f} %zu\\n", offsetof({c.__name__}, {f}));' for f, _ in c._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    got = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                                 check=True).stdout.splitlines())
    for c in structs:
        assert int(got[c.__name__]) == ctypes.sizeof(c)
        for f, _ in c._fields_:
            assert int(got[f"{c.__name__}.{f}"]) == getattr(c, f).offset, f


def test_frequencies():
    freq, mscale = ops.rope_frequencies(64, 10000.0)
    want = torch.tensor([10000.0 ** (-i / 32) for i in range(32)], dtype=torch.float64)
    assert mscale == 1.0 and torch.allclose(freq, want, rtol=1e-14, atol=0)
    stretched, mscale = ops.rope_frequencies(64, 10000.0, factor=4.0)
    assert mscale == 1.0 and torch.equal(stretched, freq / 4.0)
    blended, mscale = ops.rope_frequencies(64, 10000.0, factor=40.0, original=4096)
    assert mscale == pytest.approx(0.1 * math.log(40.0) + 1.0)
    turns = 4096 * freq / (2 * math.pi)
    # whole table entries: one entry changes the turns by 10000^(1/32)
    step = 10000.0 ** (1 / 32)
    assert torch.equal(blended[turns > 32 * step], freq[turns > 32 * step])
    assert torch.allclose(blended[turns < 1 / step], freq[turns < 1 / step] / 40, rtol=1e-14, atol=0)
    ratio = blended / freq
    # two divisions, each rounded: a ratio is off by at most 2^-52 of itself
    assert (ratio[1:] <= ratio[:-1] * (1 + 2.0 ** -51)).all() and (ratio >= (1 - 2.0 ** -52) / 40).all()
    for bad in (dict(width=3), dict(width=0), dict(width=64, base=1.0), dict(width=64, factor=0.5)):
        with pytest.raises(ValueError):
            ops.rope_frequencies(**bad)
