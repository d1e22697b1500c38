"""Backward passes that are captured while nodes of the legacy default stream live behind the moves: refused, and the process goes on.  In a process of
its own, which an error of the capture itself would end."""
import os
import subprocess
import sys

import pytest

from tests._util import ROOT

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

CODE = """
import torch
from gemmlib_b200.experts import combine_rows, gather_rows
from tests.test_experts_gpu import problem

p = problem(40, 3, 6, 200, torch.float16, 1)
order, stream = p["order"], torch.cuda.Stream()

def routed(logits):  # the leaf stands behind another operator
    return combine_rows(p["y"], order, torch.softmax(logits, -1))
def gathered(x):
    return combine_rows(gather_rows(x * 2, order), order, p["weights"])

def refused(call):
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
            call()
    except RuntimeError as e:
        assert "lives on another stream" in str(e), e
    else:
        raise AssertionError("not refused")

for make, name in ((routed, "weights"), (gathered, "x")):
    leaf = p[name].clone().requires_grad_()
    eager = make(leaf)
    torch.cuda.synchronize()
    refused(lambda: torch.autograd.grad(make(leaf), leaf, p["d_out"]))
    refused(lambda: make(leaf).backward(p["d_out"]))
    # a gradient that stops ahead of the leaf does not come to its node
    def inner():
        t = torch.softmax(leaf, -1) if make is routed else leaf * 2
        out = combine_rows(p["y"], order, t) if make is routed else combine_rows(gather_rows(t, order), order, p["weights"])
        return torch.autograd.grad(out, t, p["d_out"])[0]
    stream.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        got = inner()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, inner())
    want, = torch.autograd.grad(eager, leaf, p["d_out"])
    del eager
    # an input that was computed ahead of the capture
    t = torch.softmax(leaf, -1) if make is routed else leaf * 2
    use = (lambda t: combine_rows(p["y"], order, t)) if make is routed else (lambda t: gather_rows(t, order))
    refused(lambda: torch.autograd.grad(use(t).float().sum(), leaf))
    del t
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.autograd.grad(make(leaf), leaf, p["d_out"])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        got, = torch.autograd.grad(make(leaf), leaf, p["d_out"])
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want), name
print("ok")
"""


def test_nodes_of_the_default_stream_behind_a_captured_move():
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, env={**os.environ, "PYTHONPATH": ROOT}, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr
