"""The device error word in a process whose first call of the package is captured: it belongs to the process, not to the graph
(GPU; in a process of its own, since the word is made once)."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

SCRIPT = """
import torch
from meshy_b200.ops._ext import ext
from meshy_b200.ops.kv8 import kv8_empty
C = ext()
c = kv8_empty(8, 2, 64, 128, "cuda")
c.scale.fill_(1.0)
q = torch.randn(1, 4, 128, device="cuda").bfloat16()
bt = torch.arange(8, dtype=torch.int32, device="cuda")[None]
n = torch.full((1,), 500, dtype=torch.int32, device="cuda")
args = (q, c.k, c.v, c.scale, bt, n, 0.1)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = C.kv8_attention(*args)
assert int(C.device_error()) == 0, "not cleared before the first replay"
want = C.kv8_attention(*args)
g.replay()
assert torch.equal(out, want) and int(C.device_error()) == 0
C.kv8_attention(*args, wait=0)
g.replay()
assert int(C.device_error()) in (2, 3), "a replay cleared another call's error"
C.clear_device_error()
del g, out
torch.cuda.synchronize()
x = torch.full((1 << 20,), 7, dtype=torch.int32, device="cuda")
assert int(C.device_error()) == 0
assert torch.equal(C.kv8_attention(*args), want) and int(C.device_error()) == 0
print("right")
"""


def test_the_first_call_is_captured():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", SCRIPT], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "right" in r.stdout, r.stderr[-2000:]
