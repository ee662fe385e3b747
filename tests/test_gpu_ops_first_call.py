"""The serving operators' first calls of a process inside a stream capture: no
kernel has been loaded or launched before, and the replayed graph gives what the
calls give."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

SCRIPT = """
import sys
sys.path[:0] = [{root!r} + "/llama3.go_b200", {root!r} + "/tests"]
import numpy as np
import torch
import l3g
from ops_ref import Paged
from test_gpu_chunk_attention import Run

rng = np.random.default_rng(1)
cache = Paged(rng, [(700, 0), (90, 0)], 2, 64, True)
q = rng.normal(0, 1, (45, 4, 64)).astype(np.float32)
run = Run(l3g, cache, [40, 5], 4, q)
x = torch.randn(3, 20000, device="cuda")
y = torch.randn(3, 20001, device="cuda")  # rows off a 16-byte boundary
t = torch.zeros(3, dtype=torch.int32, device="cuda")
lp, lp2 = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
ids = torch.zeros(3, 5, dtype=torch.int32, device="cuda")
op, op2 = l3g.LogProbs(3, 20000), l3g.LogProbs(3, 20001)
pool = torch.randn(4, 256, 64, device="cuda")
src, dst = (torch.tensor([i], dtype=torch.int32, device="cuda") for i in (1, 3))

def calls(stream):
    run(stream=stream)
    op.run(x.data_ptr(), 20000, 3, t.data_ptr(), lp.data_ptr(), 0, 0, 5, ids.data_ptr(), 0, stream)
    op2.run(y.data_ptr(), 20001, 3, t.data_ptr(), lp2.data_ptr(), 0, 0, 0, 0, 0, stream)
    l3g.kv_copy_pages(pool.data_ptr(), 4, pool.data_ptr(), 4, 256, src.data_ptr(), dst.data_ptr(), 0, 1,
                      stream=stream)

g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    calls(torch.cuda.current_stream().cuda_stream)
torch.cuda.synchronize()
assert not lp.any() and torch.isnan(run.out).all() and not torch.equal(pool[1], pool[3])
g.replay()
got = [a.copy() for a in run.got()] + [a.clone() for a in (lp, lp2, ids)]
assert torch.equal(pool[1], pool[3])
run.out.fill_(float("nan")), lp.zero_(), lp2.zero_(), ids.zero_()
calls(0)
want = run.got() + [lp, lp2, ids]
for a, b in zip(got, want):
    assert np.array_equal(np.asarray(a.cpu() if hasattr(a, "cpu") else a),
                          np.asarray(b.cpu() if hasattr(b, "cpu") else b)) and a.any()
assert run.op.status() == (0, 0) and op.status() == (0, 0) and op2.status() == (0, 0)
print("same")
"""


def test_first_calls_captured(gpu_lib):
    r = subprocess.run([sys.executable, "-c", SCRIPT.format(root=ROOT)], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, CUDA_MODULE_LOADING="LAZY"))
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stdout + r.stderr[-2000:]
