"""The first calls of a process from several host threads: products and sorts that ask for different amounts of shared memory for one kernel, and plans
that ask the device how many clusters it takes."""
import os
import subprocess
import sys

import pytest

from tests._util import ROOT

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

CODE = """
import threading
import torch
from gemmlib_b200 import capi
from gemmlib_b200.experts import fp8_expert_linear, sort_by_expert
from gemmlib_b200.fp8_linear import Fp8Weight, fp8_linear
from tests.test_experts_gpu import check_order, choices_of, stack_of
from tests.test_fp8_linear_gpu import check_close, rows_of, weight_of

def product(m, k, n):
    x, w = rows_of(m, k, m), weight_of(n, k, n)
    return lambda: fp8_linear(x, w), lambda out: check_close(out, x, w)

def products(each, experts, k, n):
    x, w = rows_of(each * experts, k, 3), stack_of(experts, n, k, 4)
    offsets = torch.arange(0, each * experts + 1, each, device="cuda").int()
    def check(out):
        for e in {0, experts // 2, experts - 1}:
            at = slice(e * each, (e + 1) * each)
            check_close(out[at], type(x)(x.values[at], x.scales[at]), Fp8Weight(w.values[e], w.scales[e]))
    return lambda: fp8_expert_linear(x, w, offsets), check

def sort(tokens, experts):
    ids = choices_of(tokens, 2, experts, experts)
    return lambda: sort_by_expert(ids, experts), lambda order: check_order(order, ids, experts)

many = [(2, 9000), (1024, 128), (300, 256)]  # experts, rows of each
assert all(capi.fp8_gemm_plan(e * m, 640, 256, e)["kernel"] == "many" for e, m in many)
assert all(capi.fp8_gemm_plan(m, 512, 4096)["split"] > 1 for m in (16, 30, 60, 100))
work = [products(m, e, 256, 640) for e, m in many] + [product(m, 4096, 512) for m in (16, 30, 60, 100)] + [sort(9000, e) for e in (400, 1000, 700)]
streams = [torch.cuda.Stream() for _ in work]
torch.cuda.synchronize()
start, errors, made = threading.Barrier(len(work)), [], [None] * len(work)

def run(i):
    try:
        start.wait()
        with torch.cuda.stream(streams[i]):
            made[i] = [work[i][0]() for _ in range(10)]
    except Exception as e:
        errors.append(e)

threads = [threading.Thread(target=run, args=(i,)) for i in range(len(work))]
for t in threads: t.start()
for t in threads: t.join()
torch.cuda.synchronize()
assert not errors, errors
for (_, check), outs in zip(work, made):
    check(outs[0])
    tensors = lambda o: o if isinstance(o, tuple) else (o,)
    assert all(torch.equal(a, b) for out in outs for a, b in zip(tensors(out), tensors(outs[0])))
assert capi.last_kernel_status() == 0
print("ok")
"""


def test_first_calls_of_a_process_at_once():
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, env={**os.environ, "PYTHONPATH": ROOT}, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr
