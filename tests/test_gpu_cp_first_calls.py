"""Calls that are the first of their kind: captured into a graph in a process that has made none before; and offsets of any size, which no call has remembered."""
import math
import subprocess
import sys
import os

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

CAPTURE = """
import torch
from nccl_b200 import Communicator, get_unique_id
from nccl_b200.ops.cp import ContextParallel
torch.cuda.set_device(0)
comm = Communicator(1, 0, get_unique_id())
cp = ContextParallel(comm)
freqs = cp.rotary_frequencies(64)
for Q, K in ((1, 3000), (40, 3000), (300, 500), (2000, 2000)):
    q, k, v, dout = (torch.randn(1, n, h, 64, device="cuda").bfloat16() for n, h in ((Q, 8), (K, 2), (K, 2), (Q, 8)))
    def step():
        x, y = cp.rotary(q, q, freqs)
        out, lse = cp.attention(x, k, v, causal=True)
        delta = cp.attention_delta(dout, out)
        return (x, out, lse, delta) + cp.attention_backward(dout, x, k, v, None, lse, causal=True, delta=delta)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)), (Q, K)
    del g, got
assert comm.async_error() == 0
cp.destroy()
comm.destroy()
print("captured")
"""


def test_the_first_calls_may_be_captured():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CAPTURE], cwd=root, env=dict(os.environ, PYTHONPATH=root), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]


@pytest.mark.parametrize("Q,K", [(1, 700), (50, 60), (300, 500)])
def test_offsets_of_any_size(Q, K):
    """From keys - 1 on the first query sees all; at -queries and in front of that the last one sees none."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from nccl_b200 import Communicator, get_unique_id
    from nccl_b200.ops.cp import ContextParallel
    torch.cuda.set_device(0)
    comm = Communicator(1, 0, get_unique_id())
    cp = ContextParallel(comm)
    q, k, v = (torch.randn(2, n, 2, 64, device="cuda").bfloat16() for n in (Q, K, K))
    want = cp.attention(q, k, v)
    wants = cp.attention_backward(q, q, k, v, *want)
    for offset in (K - 1, K, K + 1, 1 << 31, (1 << 62) - 1):
        got = cp.attention(q, k, v, causal=True, offset=offset)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), offset
        assert all(torch.equal(a, b) for a, b in zip(cp.attention_backward(q, q, k, v, *got, causal=True, offset=offset), wants)), offset
    if K > 1:
        got = cp.attention(q, k, v, causal=True, offset=K - 2)
        assert not torch.equal(got[0][:, 0], want[0][:, 0]) and torch.equal(got[1][:, :, 1:], want[1][:, :, 1:])
    for offset in (-Q, -Q - 1, -(1 << 31), -(1 << 62) + 1):
        out, lse = cp.attention(q, k, v, causal=True, offset=offset)
        assert not out.any() and bool((lse == -math.inf).all())
        assert not any(bool(g.any()) for g in cp.attention_backward(q, q, k, v, out, lse, causal=True, offset=offset))
    assert bool(torch.isfinite(cp.attention(q, k, v, causal=True, offset=1 - Q)[1][:, :, -1]).all())
    torch.cuda.synchronize()
    cp.destroy()
    comm.destroy()
