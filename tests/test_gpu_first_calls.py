"""The training operators' first calls in a process, made while a CUDA graph is captured: init alone has prepared them."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import torch
from nablaengine_b200 import torch_ffi
torch_ffi.init()
assert torch_ffi._NATIVE, "init has not loaded the operators' host module"
x, g = (torch.randn(300, {cols}, device="cuda") for _ in range(2))
w, b = (torch.rand({cols}, device="cuda") for _ in range(2))
grads = [torch.randn(n, device="cuda") for n in (5000, {values})]
outs = [torch.empty_like(t) for t in grads]

def run():
    y, mean, rstd = torch_ffi.layer_norm_forward(x, w, b)
    return (y, mean, rstd, *torch_ffi.layer_norm_backward(g, x, mean, rstd, w, b),
            *torch_ffi.clip_grad_norm(grads, 1.0, out=outs), *torch_ffi.clip_grad_norm(grads[:1], 1.0, out=outs[:1]))

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = run()
graph.replay()
torch.cuda.synchronize()
captured = [t.clone() for t in (*captured, *outs)]
for a, c in zip(captured, (*run(), *outs)):
    assert torch.equal(a, c)
print("same")
"""


@pytest.mark.parametrize("cols,values", [(100, 600_000), (4096, 17), (20001, 3_000_000)])
def test_first_calls_under_capture(cols, values):
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    root = str(Path(__file__).resolve().parents[1])
    r = subprocess.run([sys.executable, "-c", PROGRAM.format(cols=cols, values=values)], cwd=root, timeout=300,
                       capture_output=True, text=True, env=dict(os.environ, PYTHONPATH=root))
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]
