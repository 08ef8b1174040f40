"""GPU tier (-m gpu): the block operators captured into a graph by a process that has called none of them before."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FIRST_USE = """
import torch
from dig_amd import ops, train

torch.set_grad_enabled(False)
bf = torch.bfloat16
g = torch.Generator(device="cuda").manual_seed(1)
rnd = lambda *shape, dtype=bf, scale=1.0: (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)
# 256x256 and 192x128 tiles (dynamic LDS above 64 KB), 64x64 tiles, k slices, packed rows, few outputs; fp32
linear = [(6272, 4096, 1024, bf), (6912, 1536, 384, bf), (5864, 81, 384, bf), (256, 256, 8192, bf), (501, 333, 777, bf), (20, 1536, 384, torch.float32), (6272, 4096, 1024, torch.float32)]
norm = [(2, 196, 384, 8, bf), (2, 20000, 64, 8, bf), (2, 300, 30, 5, torch.float32)]
lin = [(rnd(M, K, dtype=t), rnd(N, K, dtype=t, scale=K ** -0.5), rnd(N, dtype=torch.float32), rnd(M, N, dtype=t)) for M, N, K, t in linear]
gns = [(rnd(B, P, C, dtype=t), rnd(C, dtype=torch.float32), rnd(C, dtype=torch.float32), rnd(B, P, C, dtype=t), G) for B, P, C, G, t in norm]


def step():
    out = []
    for x, w, b, dy in lin:
        y, pre = ops.linear_act(x, w, b, act="gelu", res=dy, want_pre=True)
        out += [y, pre, *train.linear_act_bwd(x, w, dy, pre=pre, act="gelu")]
    for x, ga, be, dy, G in gns:
        y, mr = ops.group_norm_act(x, ga, be, groups=G, act="silu", want_stats=True)
        out += [y, mr, *train.group_norm_act_bwd(x, mr, ga, be, dy, act="silu")[:3]]
    return out


torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = step()
for k in range(3):
    for t in [v for s in lin + gns for v in s if torch.is_tensor(v)]:
        t.copy_(rnd(*t.shape, dtype=t.dtype, scale=0.5))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs, step())), k
print("captured first")
"""


def test_captured_before_any_eager_call():
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([ROOT] + [p for p in (os.environ.get("PYTHONPATH"),) if p]))
    run = subprocess.run([sys.executable, "-c", FIRST_USE], cwd=ROOT, env=env, capture_output=True, text=True, timeout=100)
    assert run.returncode == 0 and "captured first" in run.stdout, run.stderr[-3000:]
