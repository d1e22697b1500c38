"""The first calls of a process from several host threads, with rows of different widths: each asks for its own amount of shared memory."""
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

rows, widths = 700, [20488, 31744, 22528, 28672, 24000, 31000, 21008, 27000]
x = torch.randn(rows, max(widths), device="cuda").half()
made = [(torch.empty(rows, w, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")) for w in widths]
again = [(torch.empty(rows, w, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")) for w in widths]
streams = [torch.cuda.Stream() for _ in widths]
torch.cuda.synchronize()
start, errors = threading.Barrier(len(widths)), []

def work(i):
    try:
        start.wait()
        for _ in range(20):
            capi.int8_rows_quant(capi.INT8_FP16, rows, widths[i], (x, x.stride(0)), (made[i][0], widths[i]), made[i][1], streams[i].cuda_stream)
    except Exception as e:
        errors.append(e)

threads = [threading.Thread(target=work, args=(i,)) for i in range(len(widths))]
for t in threads: t.start()
for t in threads: t.join()
torch.cuda.synchronize()
assert not errors, errors
for i, w in enumerate(widths):
    capi.int8_rows_quant(capi.INT8_FP16, rows, w, (x, x.stride(0)), (again[i][0], w), again[i][1])
    torch.cuda.synchronize()
    assert torch.equal(made[i][0], again[i][0]) and torch.equal(made[i][1], again[i][1])
    top = x[:, :w].double().abs().amax(1)
    assert ((again[i][1].double() - top / 127).abs() <= top / 127 * 2.0 ** -24 * 1.01).all()
assert capi.last_kernel_status() == 0
print("ok")
"""


def test_rows_of_different_widths_at_once():
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, env={**os.environ, "PYTHONPATH": ROOT}, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr
