"""A process whose first call into the library is captured into a graph: setting up the device must
not end the capture, and replays give what plain calls give."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CHILD = """
import sys
import torch
import mensurflow_b200 as mf
n = lambda *s: torch.randn(*s, device="cuda")
x, wg, wu, wd = n(200, 130), n(130, 300) / 10, n(130, 300) / 10, n(300, 130) / 10
table, grad, ids = n(200, 64), n(5000, 64), torch.randint(0, 200, (5000,), device="cuda")

def step():
    y, saved = mf.gated_ffn(x, wg, wu, wd, save=True)
    return (y,) + mf.gated_ffn_backward(x, x, wg, wu, wd, saved=saved)

call = {
    "gemm": lambda: (mf.gemm(x, wg),),
    "few rows": lambda: (mf.gated_ffn(x[:4], wg, wu, wd),),
    "training step": step,
    "orthogonalize": lambda: (mf.orthogonalize(wg), mf.orthogonalize(x)),
    "embedding": lambda: (mf.embedding(table, ids), mf.embedding_grad(grad, ids, 200)),
}[sys.argv[1]]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = call()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, call()))
assert mf.device_status() == 0
"""


@pytest.mark.parametrize("what", ["gemm", "few rows", "training step", "orthogonalize", "embedding"])
def test_first_call_is_captured(cuda, what):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", CHILD, what], cwd=root, capture_output=True,
                          text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
