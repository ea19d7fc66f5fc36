"""Graphs that another library captures around calls of this one."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


def test_a_workspace_in_another_librarys_graph_outlives_its_growth():
    # in a process of its own, where torch is imported before the library is loaded: both then use one HIP runtime
    code = """
import numpy as np
import torch
from cgt_amd import capi, kernels as K
from cgt_amd.gpuarray import as_gpuarray
s = torch.cuda.Stream()
h = s.cuda_stream
def arrays(rows, cols):
    g = torch.Generator(device="cuda"); g.manual_seed(rows)
    x, gy = (torch.randn(rows, cols, generator=g, device="cuda") for _ in range(2))
    gamma, mean, rstd = torch.ones(cols, device="cuda"), x.mean(1), 1 / x.std(1, unbiased=False)
    outs = [torch.zeros(rows, cols, device="cuda"), torch.zeros(cols, device="cuda"), torch.zeros(cols, device="cuda")]
    return [as_gpuarray(t) for t in (x, gamma, mean, rstd, gy)], [as_gpuarray(t) for t in outs], outs
small, small_out, kept = arrays(900, 300)
large, large_out, _ = arrays(4000, 8000)
torch.cuda.synchronize()
K.layer_norm_bwd(*small, out=small_out, stream=h)
s.synchronize()
want = [t.clone() for t in kept]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=s):
    K.layer_norm_bwd(*small, out=small_out, stream=h)
K.layer_norm_bwd(*large, out=large_out, stream=h)      # the workspace grows
capi.check(capi.lib().cgt_amd_synchronize(h))           # and what it outgrew may go, unless a graph has it
fill = [torch.full((1 << 18,), 7.0, device="cuda") for _ in range(16)]
for n in range(3):
    for t in kept:
        t.zero_()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, want)), n
    assert all(bool((f == 7.0).all()) for f in fill), n
    K.layer_norm_bwd(*large, out=large_out, stream=h)
    s.synchronize()
print("replayed")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert done.returncode == 0 and "replayed" in done.stdout, done.stdout
