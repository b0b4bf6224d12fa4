"""Calls captured into a graph with guard bands around every workspace (KDEC_GUARD), which the library reads from the
environment once: a process of its own for each mode."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

TESTS = os.path.dirname(os.path.abspath(__file__))
CODE = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
from brosoundml_amd import native
from test_gpu_graph_memory import Held, capture
from test_gpu_token_graphs import same, state, work
side = torch.cuda.Stream()
ctx = native.Context(0, stream=side)
s = state(11, t=2000)
want = [t.clone() for t in work(native.Context(0), state(11, t=2000))]
torch.cuda.synchronize()
held = Held(ctx, 5000)
g, out = capture(ctx, side, s)
for _ in range(3):
    with torch.cuda.stream(side):
        g.replay()
        got = work(ctx, s)
    ctx.synchronize()
    assert same(out, want) and same(got, want)
held.free()
print("replayed")
"""


@pytest.mark.parametrize("mode", ["1", "2"])
def test_a_capture_under_guard(mode):
    code = CODE.format(root=os.path.dirname(TESTS), tests=TESTS)
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, KDEC_GUARD=mode), capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip().endswith("replayed"), r.stderr[-2000:]
    assert "guard band" not in r.stderr
