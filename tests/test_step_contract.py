"""Host validation of the step plan and the block norm (tq_step_plan_validate,
tq_block_norm_validate) and their oracles, CPU only: fake numeric addresses, the field names and
violation kinds of the other contracts."""

import ctypes
import subprocess

import numpy as np
import pytest

from conftest import ROOT

from oracle import step as ostep
from tq_mla import _abi

SHAPE, DTYPE, STRIDE, ALIGNMENT, ADDRESS, CAPACITY, SCALE, ALIAS = 1, 2, 4, 5, 6, 7, 10, 12
GiB = 1 << 30
BF, I32, F32 = _abi.DTYPE_BF16, _abi.DTYPE_I32, _abi.DTYPE_F32


def tensor(shape, dtype, address, row_stride=None):
    elem = 2 if dtype == BF else 4
    t = _abi.TqTensorSpec()
    t.rank, t.dtype, t.device_address = len(shape), dtype, address
    strides = [elem]
    for d in reversed(shape[1:]):
        strides.append(strides[-1] * d)
    strides.reverse()
    if row_stride:
        strides[0] = row_stride
    for i, (d, s) in enumerate(zip(shape, strides)):
        t.shape[i], t.strides_bytes[i] = d, s
    t.buffer_bytes = shape[0] * strides[0]
    return t


def plan(requests=5, columns=7, pool=9, tokens=30):
    s = _abi.TqStepPlanSpec()
    shapes = dict(cached_len=[requests], new_len=[requests], page_table=[requests, columns],
                  free_pages=[pool], free_count=[1], q_start=[requests + 1], kv_len=[requests],
                  seq_id=[tokens], q_pos=[tokens], slot=[tokens], free_left=[1])
    for i, (name, shape) in enumerate(shapes.items()):
        setattr(s, name, tensor(shape, I32, (i + 1) * GiB))
    return s


def norm(rows=6, width=64, kind=BF, gate=None, post=True, pre=True):
    s = _abi.TqBlockNormSpec()
    s.y = tensor([rows, width], BF, 1 * GiB)
    s.residual = tensor([rows, width], kind, 2 * GiB)
    s.out = tensor([rows, width], kind, 3 * GiB)
    if gate:
        s.gate = tensor(gate, BF, 4 * GiB)
    if post:
        s.post_weight = tensor([width], BF, 5 * GiB)
    if pre:
        s.pre_weight = tensor([width], BF, 6 * GiB)
        s.x = tensor([rows, width], BF, 7 * GiB)
    s.scale, s.post_eps, s.pre_eps = 1.0, 1e-6, 1e-6
    return s


def verdict(s):
    err = _abi.TqContractError()
    fn = _abi.lib.tq_step_plan_validate if isinstance(s, _abi.TqStepPlanSpec) else \
        _abi.lib.tq_block_norm_validate
    st = fn(ctypes.byref(s), ctypes.byref(err))
    return None if st == 0 else (err.field.decode(), st)


def test_plans_validate():
    assert verdict(plan()) is None
    assert verdict(plan(tokens=0)) is None
    assert verdict(plan(pool=0)) is None
    s = plan(); s.slot = _abi.TqTensorSpec()
    assert verdict(s) is None
    s = plan(requests=0)
    for name in ("cached_len", "new_len", "kv_len", "page_table"):
        getattr(s, name).device_address = 0
    assert verdict(s) is None


def test_plan_rejections_name_the_field_and_kind():
    for name in ("new_len", "kv_len", "q_start", "q_pos", "slot", "free_count", "free_left"):
        s = plan(); getattr(s, name).shape[0] += 1
        assert verdict(s) == (name, SHAPE), name
    for name in ("cached_len", "new_len", "page_table", "free_pages", "free_count", "q_start",
                 "kv_len", "seq_id", "q_pos", "slot", "free_left"):
        s = plan(); getattr(s, name).dtype = F32
        assert verdict(s) == (name, DTYPE), name
        s = plan(); getattr(s, name).device_address = 0
        assert verdict(s) == (name, ADDRESS), name
        s = plan(); getattr(s, name).device_address += 2
        assert verdict(s) == (name, ALIGNMENT), name
        s = plan(); getattr(s, name).buffer_bytes -= 4
        assert verdict(s) == (name, CAPACITY), name
    s = plan(); s.page_table.strides_bytes[0] += 4
    assert verdict(s) == ("page_table", STRIDE)
    s = plan(); s.page_table.rank = 1
    assert verdict(s) == ("page_table", SHAPE)


@pytest.mark.parametrize("out", ["page_table", "q_start", "kv_len", "seq_id", "q_pos", "slot",
                                 "free_left"])
@pytest.mark.parametrize("other", ["cached_len", "new_len", "free_pages", "free_count"])
def test_plan_outputs_never_overlap_an_input(out, other):
    s = plan()
    getattr(s, out).device_address = getattr(s, other).device_address
    assert verdict(s) == (out, ALIAS)


def test_norms_validate():
    for kind in (BF, F32):
        for gate in (None, [64], [6, 64]):
            for post in (False, True):
                for pre in (False, True):
                    assert verdict(norm(kind=kind, gate=gate, post=post, pre=pre)) is None
    assert verdict(norm(rows=0)) is None
    assert verdict(norm(width=32768)) is None
    s = norm(); s.out.device_address = s.residual.device_address
    assert verdict(s) is None                                   # the residual updated in place
    s.x.device_address = s.y.device_address
    assert verdict(s) is None                                   # x written over y
    s = norm(); s.y = tensor([6, 64], BF, 1 * GiB, row_stride=160)
    assert verdict(s) is None


def test_norm_rejections_name_the_field_and_kind():
    assert verdict(norm(width=60)) == ("y", SHAPE)
    assert verdict(norm(width=32776)) == ("y", SHAPE)
    assert verdict(norm(kind=I32)) == ("residual", DTYPE)
    s = norm(); s.out.dtype = F32
    assert verdict(s) == ("out", DTYPE)
    assert verdict(norm(gate=[32])) == ("gate", SHAPE)
    assert verdict(norm(gate=[5, 64])) == ("gate", SHAPE)
    s = norm(); s.post_weight.shape[0] = 32
    assert verdict(s) == ("post_weight", SHAPE)
    s = norm(); s.x = _abi.TqTensorSpec()
    assert verdict(s) == ("x", SHAPE)
    s = norm(); s.pre_weight = _abi.TqTensorSpec()
    assert verdict(s) == ("x", SHAPE)
    for name in ("y", "residual", "out", "x"):
        s = norm(); getattr(s, name).device_address += 8
        assert verdict(s) == (name, ALIGNMENT), name
        s = norm(); t = getattr(s, name); t.strides_bytes[0] += 8; t.buffer_bytes += 64
        assert verdict(s) == (name, STRIDE), name
    for name in ("post_weight", "pre_weight"):
        s = norm(); getattr(s, name).device_address += 8
        assert verdict(s) == (name, ALIGNMENT), name
    s = norm(); s.scale = float("inf")
    assert verdict(s) == ("scale", SCALE)
    s = norm(); s.post_eps = 0.0
    assert verdict(s) == ("post_eps", SCALE)
    s = norm(); s.pre_eps = float("nan")
    assert verdict(s) == ("pre_eps", SCALE)


def test_norm_outputs_overlap_nothing_but_their_own_place():
    s = norm(); s.out.device_address = s.y.device_address
    assert verdict(s) == ("out", ALIAS)
    s = norm(); s.out.device_address = s.residual.device_address + 128
    assert verdict(s) == ("out", ALIAS)                         # shifted by one row
    s = norm(); s.x.device_address = s.residual.device_address
    assert verdict(s) == ("x", ALIAS)
    s = norm(); s.x.device_address = s.out.device_address
    assert verdict(s) == ("x", ALIAS)
    s = norm(gate=[6, 64]); s.x.device_address = s.gate.device_address
    assert verdict(s) == ("x", ALIAS)
    s = norm(); s.out.device_address = s.pre_weight.device_address
    assert verdict(s) == ("out", ALIAS)


def test_plan_oracle_on_a_hand_written_step():
    # request 0 grows inside its page, 1 starts empty and takes two, 2 idles, 3 crosses a border
    table = np.full((4, 3), -1)
    table[0, 0], table[2, 0], table[3, 0] = 8, 9, 10
    got = ostep.step_plan([10, 0, 5, 63], [2, 65, 0, 3], table, [4, 5, 6, 7], 4, 75)
    q_start, kv_len, seq_id, q_pos, slot, out, left, flags = got
    assert q_start.tolist() == [0, 2, 67, 67, 70] and kv_len.tolist() == [12, 65, 5, 66]
    assert out.tolist() == [[8, -1, -1], [7, 6, -1], [9, -1, -1], [10, 5, -1]] and left == 1 and flags == 0
    assert slot[:2].tolist() == [8 * 64 + 10, 8 * 64 + 11] and slot[66] == 6 * 64
    assert q_pos[67:].tolist() == [63, 64, 65, -1, -1, -1, -1, -1]
    assert slot[67:70].tolist() == [10 * 64 + 63, 5 * 64, 5 * 64 + 1] and seq_id[69] == 3


def test_norm_oracle_without_its_parts_is_a_sum():
    rng = np.random.default_rng(0)
    y, h = rng.standard_normal((2, 3, 16))
    out, x = ostep.block_norm(y, h, scale=0.5)
    assert x is None and np.array_equal(out, h + 0.5 * y)
    out, x = ostep.block_norm(y, h, pre_weight=np.ones(16), post_weight=np.ones(16), eps=1e-12)
    np.testing.assert_allclose((x * x).mean(axis=1), 1.0, rtol=1e-9)
    np.testing.assert_allclose(((out - h) ** 2).mean(axis=1), 1.0, rtol=1e-9)


def test_struct_layout_matches_a_c_compiler(tmp_path):
    structs = {name: getattr(_abi, name) for name in ("TqStepPlanSpec", "TqBlockNormSpec", "TqMlaChunkSpec")}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT / "include" / "tq_mla.h"}"', "int main(){"]
    for name, cls in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for name, cls in structs.items():
        assert int(got[name]) == ctypes.sizeof(cls), name
        for f, _ in cls._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(cls, f).offset, (name, f)
