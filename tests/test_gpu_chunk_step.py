"""GPU: the operators of a prefill step together, as a serving loop runs them: the step plan from the
request lengths, the norm in front of the block, the prologue without absorption, the chunk
attention over the rows it wrote, and the step between this block and the next. Two steps of the
same requests, so that the second one attends over rows of the first.

The chain is checked stage by stage on the device's own inputs to each stage (the plan exactly, the
others against their float64 oracles at the tolerances of their own tests), which is what makes the
bounds tight; and the attention's output against the absorbed attention of this library on the same
rows, whose queries and outputs carry the key and value weights instead."""

import numpy as np
import pytest
import torch

from oracle import chunk as ochunk
from oracle import prologue as opro
from oracle import step as ostep
from test_gpu_prologue import _check_q
from test_gpu_step import _check_norm
from tq_mla import _abi, ops

pytestmark = pytest.mark.gpu
ROW = {_abi.KV_BF16: 1024, _abi.KV_FP8_E4M3: 544, _abi.KV_BF16_ROPE576: 1152}


def bf16(a, device):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(torch.bfloat16).to(device)


def f64(t):
    return t.double().cpu().numpy()


@pytest.mark.parametrize("fmt,heads,dn,dr", [(_abi.KV_BF16_ROPE576, 16, 128, 64), (_abi.KV_FP8_E4M3, 8, 256, 0)])
def test_two_prefill_steps(cuda_device, fmt, heads, dn, dr):
    dev = cuda_device
    rng = np.random.default_rng(fmt)
    dm, rq, dv, requests, slots = 512, 256, dn, 4, 8
    w = {k: bf16(v, dev) for k, v in dict(
        w_qa=rng.standard_normal((rq, dm)) / np.sqrt(dm), q_norm=rng.uniform(0.5, 1.5, rq),
        w_qb=rng.standard_normal((heads * (dn + dr), rq)) / np.sqrt(rq),
        w_kva=rng.standard_normal((512 + dr, dm)) / np.sqrt(dm), kv_norm=rng.uniform(0.5, 1.5, 512),
        w_uk=rng.standard_normal((heads, dn, 512)) / np.sqrt(512),
        w_uv=rng.standard_normal((heads, dv, 512)) / np.sqrt(512),
        w_o=rng.standard_normal((dm, heads * dv)) / np.sqrt(heads * dv),
        pre=rng.uniform(0.5, 1.5, dm), post=rng.uniform(0.5, 1.5, dm), gate=rng.uniform(-1, 1, dm)).items()}
    pool = torch.full((requests * slots, 64, ROW[fmt]), 255, dtype=torch.uint8, device=dev)
    table = torch.full((requests, slots), -1, dtype=torch.int32, device=dev)
    free = torch.from_numpy(rng.permutation(requests * slots).astype(np.int32)).to(dev)
    count = torch.tensor([requests * slots], dtype=torch.int32, device=dev)
    cached = torch.zeros(requests, dtype=torch.int32, device=dev)
    scale = (dn + dr) ** -0.5
    flags = torch.zeros(1, dtype=torch.int32, device=dev)
    for lengths in ([130, 1, 64, 40], [1, 200, 0, 77]):
        tokens = sum(lengths)
        new = torch.tensor(lengths, dtype=torch.int32, device=dev)
        before = table.cpu().numpy().copy()
        plan = ops.step_plan(cached, new, table, free, count, tokens=tokens, flags=flags)
        want = ostep.step_plan(cached.tolist(), lengths, before, free.tolist(), int(count), tokens)
        for name, ref in zip(("q_start", "kv_len", "seq_id", "q_pos", "slot", "page_table"), want):
            np.testing.assert_array_equal(getattr(plan, name).cpu().numpy(), ref, err_msg=name)

        residual = torch.from_numpy(rng.standard_normal((tokens, dm)).astype(np.float32)).to(dev)
        block_in = bf16(rng.standard_normal((tokens, dm)), dev)
        hidden, x = ops.block_norm(block_in, residual, gate=w["gate"], scale=0.5, pre_weight=w["pre"])
        _check_norm({"y": block_in, "residual": residual, "gate": w["gate"], "post_weight": None,
                     "pre_weight": w["pre"]}, hidden, x, 0.5)

        q = ops.mla_prologue(x, w["w_qa"], w["q_norm"], w["w_qb"], None, w["w_kva"], w["kv_norm"],
                             plan.q_pos, plan.seq_id, plan.page_table, pool, heads=heads, nope_dim=dn,
                             rope_dim=dr, kv_format=fmt, flags=flags)
        cq = opro.bf16(f64(x) @ f64(w["w_qa"]).T)
        qf = opro.bf16(opro.rms_norm(cq, f64(w["q_norm"]), 1e-6) @ f64(w["w_qb"]).T).reshape(tokens, heads, -1)
        if dr:
            qf[:, :, dn:] = opro.rope(qf[:, :, dn:], plan.q_pos.cpu().numpy(), 10000.0)
        _check_q(f64(q), qf)

        out, lse = ops.mla_chunk(q, w["w_uk"], w["w_uv"], pool, plan.page_table, plan.q_start, plan.q_pos,
                                 plan.kv_len, scale=scale, max_keys=requests * slots * 64, kv_format=fmt)
        with np.errstate(invalid="ignore"):
            rows = ochunk.pool_rows(pool.reshape(-1, ROW[fmt]).cpu().numpy(), fmt)
        ref, ref_lse = ochunk.chunk_attention(
            f64(q), f64(w["w_uk"]), f64(w["w_uv"]), rows, plan.page_table.cpu().numpy(),
            plan.q_start.cpu().numpy(), plan.q_pos.cpu().numpy(), plan.kv_len.cpu().numpy(), scale=scale)
        assert np.linalg.norm(f64(out) - ref) <= 1e-2 * np.linalg.norm(ref)
        assert np.abs(f64(lse) - ref_lse).max() <= 2e-2

        if fmt == _abi.KV_BF16_ROPE576:
            # the absorbed form: w_uk folded into the query, w_uv applied to its latent output
            q_abs = torch.cat([torch.einsum("thd,hdr->thr", q[:, :, :dn].float(), w["w_uk"].float()),
                               q[:, :, dn:].float()], dim=2).to(torch.bfloat16)
            lat, lat_lse = ops.mla_decode(q_abs, pool, plan.page_table, plan.seq_id, plan.q_pos, plan.kv_len,
                                          scale=scale, query_counts=lengths, prefill=True)
            folded = torch.einsum("thr,hvr->thv", lat.float(), w["w_uv"].float())
            assert float((folded - out.float()).norm() / folded.norm()) <= 1e-2
            assert float((lat_lse - lse).abs().max()) <= 2e-2

        y = (out.reshape(tokens, -1).float() @ w["w_o"].float().T).to(torch.bfloat16)
        after, x_next = ops.block_norm(y, hidden, post_weight=w["post"], pre_weight=w["pre"], scale=1.0)
        _check_norm({"y": y, "residual": hidden, "gate": None, "post_weight": w["post"],
                     "pre_weight": w["pre"]}, after, x_next, 1.0)
        assert int(flags) == 0
        cached, count = plan.kv_len.clone(), plan.free_left.clone()
