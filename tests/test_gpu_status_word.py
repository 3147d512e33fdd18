"""The status word of a process whose first call is captured: it belongs to no graph."""
import subprocess
import sys
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import torch
import rtx_b200
from rtx_b200 import ops

dev = torch.device("cuda", 0)
x = torch.ones(64, 96, device=dev, dtype=torch.bfloat16)
w = torch.ones(3, 128, 96, device=dev, dtype=torch.bfloat16)
good = torch.tensor([0, 10, 20, 64], dtype=torch.int32, device=dev)
bad = torch.tensor([0, 40, 20, 64], dtype=torch.int32, device=dev)
want = torch.full((64, 128), 96.0, device=dev, dtype=torch.bfloat16)

def reported():
    try:
        ops.check_device_status(dev)
    except RuntimeError as e:
        assert "offsets" in str(e), e
        return True
    return False

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = rtx_b200.mxfp8_grouped_linear(x, w, good)           # the process's first call
assert ops.status_word(dev).item() == 0                     # set before any replay
for _ in range(2):
    rtx_b200.mxfp8_grouped_linear(x, w, bad)                # reports, beside the graph
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    assert reported()                                       # the replay has not cleared it
    assert not reported()
good.copy_(bad)
graph.replay()
assert reported()                                           # and a replayed call reports into the same word
del graph, y
print("word ok")
"""


def test_a_captured_first_call_leaves_the_word_outside_the_graph(native_lib):
    done = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "word ok" in done.stdout, done.stdout[-2000:] + done.stderr[-2000:]
