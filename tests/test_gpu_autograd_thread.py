"""The operator's backward as the first CUDA work of autograd's thread, in a
process of its own: the incoming gradients are given as they are, so that no
torch kernel runs on that thread before the solver's."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import sys
sys.path[:0] = [{root!r}, {pkg!r}]
import torch
import ilqr_workload as wl
import mpc_compat
B, T = 7, 4
inp = wl.make_inputs(B, T, seed=0)
t = lambda a: torch.from_numpy(a).to("cuda:0")
C = t(inp["C"]).permute(1, 0, 2, 3).contiguous().requires_grad_(True)
c = t(inp["c"]).permute(1, 0, 2).contiguous()
x, u, _ = mpc_compat.MPC(10, 4, T, lqr_iter=2)(t(inp["x0"]), mpc_compat.QuadCost(C, c), type("Dx", (), dict(dt=0.05))())
gX, gU = (t(g).permute(1, 0, 2) for g in wl.make_backward_seeds(B, T))
torch.autograd.backward([x, u], [gX, gU])
assert torch.isfinite(C.grad).all() and C.grad.abs().sum() > 0
"""


def test_backward_is_the_first_cuda_work_of_its_thread():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", PROGRAM.format(root=root, pkg=os.path.join(root, "ca-ac-mpc_b200"))],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
