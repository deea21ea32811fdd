"""GPU test of the 8-bit cache attention's very first calls in a process, from
several host threads at once (the calls release the interpreter lock): each has
to find the kernels' shared-memory limits set."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import sys, threading
import torch
from ssd import ops

dtype, hd, n = getattr(torch, sys.argv[1]), int(sys.argv[2]), 8
H, Hkv, slots, T = 8, 2, 700, 5
g = torch.Generator("cuda").manual_seed(1)
codes = torch.randint(0, 127, (2, Hkv, slots, hd), generator=g, device="cuda").to(torch.uint8).view(torch.float8_e4m3fn)
scales = torch.full((2, Hkv, slots), 120, dtype=torch.uint8, device="cuda")
layer = ops.KVLayerQ8(codes[0], codes[1], scales[0], scales[1])
q = torch.randn(T, H * hd, generator=g, device="cuda").to(dtype)
plen = torch.full((T,), slots, dtype=torch.int32, device="cuda")
jobs = [(torch.cuda.Stream(), ops.Workspace(torch.device("cuda"), 16, 16), torch.zeros_like(q)) for _ in range(n)]
torch.cuda.synchronize()
start, errors = threading.Barrier(n), []

def call(stream, ws, out):
    with torch.cuda.stream(stream):
        start.wait(60)
        try:
            ops.tree_attention_q8(q, layer, H, Hkv, hd, plen, out, ws)
        except Exception as e:
            errors.append(e)

threads = [threading.Thread(target=call, args=j) for j in jobs]
for t in threads:
    t.start()
for t in threads:
    t.join()
torch.cuda.synchronize()
assert not errors, errors
for _, ws, out in jobs:
    ws.check_status()
    assert torch.equal(out, jobs[0][2]) and bool(out.abs().sum() > 0)
print("ok")
"""


@pytest.mark.parametrize("dtype,hd", [("bfloat16", 128), ("bfloat16", 64), ("bfloat16", 112), ("float32", 128)])
def test_first_calls_from_many_threads(dtype, hd):
    env = dict(os.environ, PYTHONPATH=os.path.join(ROOT, "subnetwork-speculative-decoding_b200"))
    r = subprocess.run([sys.executable, "-c", PROGRAM, dtype, str(hd)], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr[-2000:]
