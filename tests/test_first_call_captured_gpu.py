"""The first call on a device may be one that a CUDA graph records."""
import subprocess
import sys

import pytest

from tests.conftest import ROOT

pytestmark = pytest.mark.gpu

PROGRAM = """
import torch
from eraserdit_b200 import _native
from eraserdit_b200.block_topk import block_topk_attention
from eraserdit_b200.linear import linear_act, linear_bf16

x = torch.randn(256, 256, device="cuda").bfloat16()
w = torch.randn(256, 256, device="cuda").bfloat16()
q = torch.randn(1, 256, 2, 64, device="cuda").bfloat16()
device = x.device


def first():
    return linear_bf16(x, w)


def second():
    return linear_act(x, w, activation="silu"), block_topk_attention(q, q, q, 0.125, 2)


outs = []
for call in (first, second):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    outs.append((graph, out))
# before any replay: what the captured kernels will report to reads as nothing yet, and
# calls outside a graph do not depend on it
assert _native.read_status(device) == 0
eager = [first(), second()]
x.mul_(0.5)
q.neg_()
for graph, _ in outs:
    graph.replay()
assert torch.equal(outs[0][1], first())
assert all(torch.equal(a, b) for a, b in zip(outs[1][1], second()))
assert not torch.equal(eager[0], outs[0][1])
assert _native.read_status(device) == 0
# a timeout of a captured kernel is seen, and cleared
words = _native._captured_status[device.index]
assert words and all(t is not _native._status[device.index] for t in words)
words[0].fill_(4)
assert _native.read_status(device) == 4 and _native.read_status(device) == 0
# graphs recorded from now on use the device's word
n = len(words)
with torch.cuda.graph(torch.cuda.CUDAGraph()):
    second()
assert len(words) == n
"""


def test_first_call_in_a_capture():
    done = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-3000:]
