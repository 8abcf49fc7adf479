"""GPU: the first calls of a process: inside a capture, and from several host threads at once."""

import os
import subprocess
import sys

import pytest

from conftest import PKG, ROOT

pytestmark = pytest.mark.gpu

MADE = """
import threading
import torch
from tq_mla import ops

dev = torch.device("cuda", 0)
g = torch.Generator(device=dev).manual_seed(3)
t, n, heads, k = 5, 300, 64, 20
table = torch.randperm(8, generator=g, device=dev).int()[None]
index = torch.zeros((8, 64, 144), dtype=torch.uint8, device=dev)
q = torch.randn((t, heads, 128), generator=g, device=dev).bfloat16()
keys = torch.randn((n, 128), generator=g, device=dev).bfloat16()
w = torch.randn((t, heads), generator=g, device=dev)
seq, pos = torch.zeros(n, dtype=torch.int32, device=dev), torch.arange(n, dtype=torch.int32, device=dev)
kv_len = torch.tensor([n], dtype=torch.int32, device=dev)

def buffers():
    return [torch.zeros((t, heads, 128), dtype=torch.uint8, device=dev), torch.zeros((t, heads), device=dev),
            torch.full((t, 512), float("-inf"), device=dev), torch.zeros((t, k), dtype=torch.int32, device=dev),
            torch.zeros(t, dtype=torch.int32, device=dev), torch.zeros((t, 4), dtype=torch.int32, device=dev),
            torch.zeros(t, dtype=torch.int32, device=dev), index.clone()]

def calls(b):
    codes, w8, scores, idx, length, pages, rows, cache = b
    s, p = seq[-t:], pos[-t:]
    return [ops.IndexWrite(None, keys, None, table, seq, pos, cache, None, None),
            ops.IndexWrite(q, keys[-t:], w, table, s, p, cache, codes, w8),
            ops.IndexScores(codes, w8, cache, table, s, p, kv_len, scores),
            ops.IndexSelect(scores, s, p, kv_len, idx, length),
            ops.IndexSelect(scores, s, p, kv_len, pages, rows, page_table=table, keep_last=1)]

def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))

"""
CAPTURED = MADE + """
b = buffers()
run = calls(b)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    for call in run:
        call()
graph.replay()
torch.cuda.synchronize()
b2 = buffers()
for call in calls(b2):
    call()
torch.cuda.synchronize()
assert same(b, b2) and int(b[4].min()) == k and bool(torch.isfinite(b[2][:, :296]).all())
del graph
print("same")
"""
THREADS = MADE + """
made = [buffers() for _ in range(6)]
streams = [torch.cuda.Stream() for _ in made]
torch.cuda.synchronize()
failed = []

def work(b, stream):
    try:
        with torch.cuda.stream(stream):
            for _ in range(20):
                for call in calls(b):
                    call()
    except Exception as e:
        failed.append(e)

threads = [threading.Thread(target=work, args=x) for x in zip(made, streams)]
for x in threads:
    x.start()
for x in threads:
    x.join()
torch.cuda.synchronize()
assert not failed, failed
assert all(same(made[0], b) for b in made) and int(made[0][4].min()) == k
print("same")
"""


@pytest.mark.parametrize("program", [CAPTURED, THREADS], ids=["captured", "threads"])
def test_first_calls_of_a_process(cuda_device, program):
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([str(PKG), str(ROOT)]))
    r = subprocess.run([sys.executable, "-c", program], env=env, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]
