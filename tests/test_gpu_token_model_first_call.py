"""The first call that a process makes of an operator may be one that a CUDA graph captures."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = """
import sys
sys.path.insert(0, {package!r})
import torch
import pararnn_b200 as prb
torch.manual_seed(0)
q, k, v = (torch.randn(2, 1500, 2, 64, device="cuda").bfloat16() for _ in range(3))
g = torch.tensor([-0.1, -0.2], device="cuda")
x, w, ids = torch.randn(5, 7, 64, device="cuda"), torch.randn(9, 64, device="cuda"), torch.arange(9, device="cuda")
pool = torch.randn(2, 2, 64, 64, device="cuda")
calls = {{
    "attention": lambda: prb.linear_attention(q, k, v, g, return_state=True),
    "step": lambda: (prb.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, pool.clone()),),
    "norm": lambda: (prb.group_norm(x, 4, activation="silu"),),
    "embedding": lambda: (prb.embedding(ids, w, 2.0),),
}}
call = calls[{name!r}]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph), torch.no_grad():
    got = call()
graph.replay()
torch.cuda.synchronize()
with torch.no_grad():
    want = call()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("same")
"""


@pytest.mark.parametrize("name", ["attention", "step", "norm", "embedding"])
def test_a_captured_first_call(name):
    program = PROGRAM.format(package=os.path.join(ROOT, "pararnn-torch_b200"), name=name)
    r = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]
