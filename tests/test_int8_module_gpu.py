"""Int8Linear and RMSNormInt8 as modules, and the int8 operators run together: a feed-forward block, a stack in a CUDA graph."""
import copy

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def normal(*shape, dtype=torch.float16, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def same(a, b):
    assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("k", [512, 500, 7])
def test_module_is_its_operators(k, dtype):
    from gemmlib_b200.int8_linear import Int8Linear, Int8Rows, int8_linear, quantize_int8

    w, bias, x = normal(96, k, dtype=dtype, scale=0.1), normal(96, dtype=dtype, seed=1), normal(2, 5, k, dtype=dtype, seed=2)
    rows = quantize_int8(w)
    for b in (None, bias, bias.float()):
        layer = Int8Linear(w, b)
        want = int8_linear(quantize_int8(x), rows, None if b is None else b.to(dtype), dtype=dtype)
        for _ in range(3):  # the weights are fetched early from the second call on
            same(layer(x), want)
        same(layer(quantize_int8(x)), want)
        out = torch.empty_like(want)
        assert layer(x, out=out).data_ptr() == out.data_ptr()
        same(out, want)
        same(Int8Linear.from_rows(rows, b, dtype)(x), want)
        same(Int8Linear.from_rows(Int8Rows(rows.values.contiguous(), rows.scales), b, dtype)(x), want)
        same(copy.deepcopy(layer)(x), want)
        other = Int8Linear(torch.zeros_like(w), b)
        other(x)
        other.load_state_dict(layer.state_dict())
        same(other(x), want)
        same(layer.cpu().cuda()(x), want)


def test_a_copy_waits_for_its_weights():
    from gemmlib_b200.int8_linear import Int8Linear

    layer, x = Int8Linear(normal(96, 512)), normal(2, 512, seed=2)
    want = layer(x)
    assert layer._settled
    other = copy.deepcopy(layer)
    assert not other._settled
    same(other(x), want)


def test_an_output_of_another_type_than_the_weights():
    from gemmlib_b200.int8_linear import Int8Linear, quantize_int8

    layer, x = Int8Linear(normal(32, 64)), normal(3, 64, seed=1)
    out = torch.empty(3, 32, dtype=torch.bfloat16, device="cuda")
    rows = quantize_int8(x)
    layer(rows, out=out)
    same(layer(x.bfloat16()), Int8Linear.from_rows(quantize_int8(normal(32, 64)))(x.bfloat16()))
    assert (out.float() - layer(rows).float()).abs().max() <= 2.0 ** -8 * 1.01 * layer(rows).float().abs().max() + 2.0 ** -24


def test_a_model_converted_to_another_type_keeps_its_scales():
    from gemmlib_b200.int8_linear import Int8Linear

    layer, x = Int8Linear(normal(32, 64), normal(32, seed=2)), normal(3, 64, seed=1)
    want = layer(x)
    same(copy.deepcopy(layer).half()(x), want)
    other = copy.deepcopy(layer).to(torch.bfloat16)
    assert other.q_scales.dtype == torch.float32 and torch.equal(other.q_scales, layer.q_scales)
    same(other(x), want)


@pytest.mark.parametrize("rows", [1, 40])
def test_forward_right_behind_the_quantization(rows):
    """The weights of a second forward are fetched early: not before the quantizer ahead of the first one is done."""
    from gemmlib_b200.int8_linear import Int8Linear, Int8Rows

    w, x = normal(8192, 4096, seed=1, scale=0.02), normal(rows, 4096, seed=2)
    want = Int8Linear(w)(x)
    torch.cuda.synchronize()
    for _ in range(10):
        layer = Int8Linear(w)  # into memory that another layer's weights were in
        first, second = layer(x), layer(x)
        same(first, want), same(second, want)
        layer.q_weights.zero_()
        del layer


def test_first_calls_of_a_process_inside_a_capture():
    import os
    import subprocess
    import sys

    from tests._util import ROOT

    code = """
import torch
from gemmlib_b200.int8_linear import Int8Rows, int8_linear, quantize_int8, rms_norm_int8, silu_mul_int8
g = torch.Generator(device="cuda").manual_seed(0)
made = []
for m, k, n in ((1, 512, 256), (16, 4096, 512), (300, 1024, 256), (600, 256, 4096)):
    x = torch.randn(m, k, generator=g, device="cuda").half()
    q = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    made.append((x, Int8Rows(q, torch.full((n,), 1e-3, device="cuda"))))
wide = torch.randn(700, 40000, generator=g, device="cuda").half()
def run():
    out = []
    for x, w in made:
        rows, h = rms_norm_int8(x, x[0], residual=x)
        out += [int8_linear(rows, w), h, silu_mul_int8(x, x).dequantize(), quantize_int8(x).dequantize()]
    return out + [quantize_int8(wide).dequantize(), quantize_int8(wide[:, :20000]).dequantize()]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(captured, run()))
print("ok")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env={**os.environ, "PYTHONPATH": ROOT}, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr


def test_gradients_are_refused():
    from gemmlib_b200.int8_linear import Int8Linear, RMSNormInt8, rms_norm_int8

    layer, x = Int8Linear(normal(32, 64)), normal(3, 64, seed=1).requires_grad_()
    norm = RMSNormInt8(normal(64, seed=2))
    for call in (lambda: layer(x), lambda: norm(x), lambda: norm(x.detach(), residual=x),
                 lambda: rms_norm_int8(x.detach(), normal(64).requires_grad_())):
        with pytest.raises(RuntimeError, match="no backward pass"):
            call()
    with torch.no_grad():
        layer(x), norm(x)
    assert not any(p.requires_grad for p in [*layer.parameters(), *norm.parameters()])


@pytest.mark.parametrize("rows", [1, 3, 40, 700])
def test_feed_forward_block(rows):
    """The whole chain, many times over and in a graph, gives the bits of its calls one by one with a wait after each; the waits
    between its kernels are their own (programmatic launches), so a missing one would show here."""
    from gemmlib_b200 import capi
    from gemmlib_b200.int8_linear import Int8Linear, RMSNormInt8, silu_mul_int8

    hidden, ffn = 512, 1408
    x, residual = normal(rows, hidden, seed=1), normal(rows, hidden, seed=2)
    norm = RMSNormInt8(normal(hidden, seed=3))
    gate_up, down = Int8Linear(normal(2 * ffn, hidden, seed=4, scale=0.05)), Int8Linear(normal(hidden, ffn, seed=5, scale=0.05))

    def block(x, residual, wait=lambda: None):
        wait()
        a, h = norm(x, residual)
        wait()
        both = gate_up(a)
        wait()
        a = silu_mul_int8(both[:, :ffn], both[:, ffn:])
        wait()
        return down(a), h

    want, h = block(x, residual, torch.cuda.synchronize)
    torch.cuda.synchronize()
    # the definition in 64 bits, from the rows that were multiplied
    a, _ = norm(x, residual)
    both = gate_up(a)
    g, u = both[:, :ffn].double(), both[:, ffn:].double()
    acts = silu_mul_int8(both[:, :ffn], both[:, ffn:])
    exact = ((acts.values.double() @ down.q_weights.double().t()) * acts.scales.double()[:, None] * down.q_scales.double())
    assert ((want.double() - exact).abs() <= exact.abs() * (2.0 ** -11 + 2.0 ** -21) + 2.0 ** -25).all()
    assert ((acts.dequantize().double() - g * torch.sigmoid(g) * u).abs()
            <= acts.scales.double()[:, None] * (0.5 + 127 * 2.0 ** -11 + 0.01)).all()  # half a step, and a rounding to fp16
    for _ in range(20):
        outs = [block(x, residual) for _ in range(5)]
    for o, r in outs:
        same(o, want), same(r, h)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = block(x, residual)
        second = block(first[0], first[1])
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    same(first[0], want), same(first[1], h)
    o, r = block(want, h, torch.cuda.synchronize)
    same(second[0], o), same(second[1], r)
    assert capi.last_kernel_status() == 0


@pytest.mark.parametrize("rows", [1, 17, 300])
def test_int8_stack_is_its_calls_one_by_one(rows):
    from gemmlib_b200.int8_linear import quantize_int8, silu_mul_int8
    from gemmlib_b200.stack import llama_like_int8_stack

    hidden, ffn = 256, 704
    stack = llama_like_int8_stack(hidden, ffn, 2, "cuda", seed=3)
    assert stack.num_linears == 14
    assert stack.weight_bytes() == 2 * (4 * hidden * hidden + 3 * hidden * ffn + 4 * (5 * hidden + 2 * ffn))
    x = normal(rows, hidden, seed=4)
    bufs = {"x": x.clone()}
    for i in (0, 7):
        q, k, v, o, gate, up, down = (layer for layer, _, _ in stack.steps[i:i + 7])
        a = stack.int8_inputs[i](bufs)
        bufs["q"], bufs["k"], bufs["v"] = q(a), k(a), v(a)
        bufs["o"] = o(quantize_int8(bufs["q"]))
        a = stack.int8_inputs[i + 4](bufs)
        bufs["gate"], bufs["up"] = gate(a), up(a)
        bufs["down"] = down(silu_mul_int8(bufs["gate"], bufs["up"]))
    want = bufs["x"] + bufs["down"]
    for _ in range(3):
        same(stack.forward(x, "x"), want)
        for name in ("q", "k", "v", "o", "gate", "up", "down"):
            same(stack.buffers(rows)[name], bufs[name])


def test_int8_and_int4_layers_in_one_stack():
    """Rows of a buffer are shared as long as it is not written, by a step or by a hook."""
    from gemmlib_b200.int8_linear import Int8Linear
    from gemmlib_b200.ms_blkq4linear import BlkQ4Linear
    from gemmlib_b200.stack import LinearStack

    i8 = [Int8Linear(normal(128, 128, seed=s, scale=0.1)) for s in range(4)]
    i4 = BlkQ4Linear(64, True, True, normal(128, 128, seed=9, scale=0.1))
    steps = [(i8[0], "x", "a"), (i8[1], "x", "b"), (i4, "a", "x2"), (i8[2], "x2", "a"), (i8[3], "a", "c"), (i8[0], "a", "a"),
             (i8[1], "a", "d"), (i4, "d", "e")]
    stack = LinearStack(steps, between={4: lambda bufs: bufs["a"].mul_(2)})
    x = normal(5, 128, seed=10)
    bufs = {"x": x}
    for n, (layer, src, dst) in enumerate(steps):
        bufs[dst] = layer(bufs[src].clone())
        if n == 4:
            bufs["a"] = bufs["a"] * 2
    for _ in range(2):
        same(stack.forward(x, "e"), bufs["e"])
        for name in "abcd":
            same(stack.buffers(5)[name], bufs[name])


def test_stack_refuses_int8_inputs_of_other_steps():
    from gemmlib_b200.int8_linear import Int8Linear, quantize_int8
    from gemmlib_b200.ms_blkq4linear import BlkQ4Linear
    from gemmlib_b200.stack import LinearStack

    i4, i8 = BlkQ4Linear(64, True, True, normal(128, 128, scale=0.1)), Int8Linear(normal(128, 128))
    for bad in (0, 2, -1):
        with pytest.raises(ValueError, match="which has no Int8Linear"):
            LinearStack([(i4, "x", "a"), (i8, "a", "b")], int8_inputs={bad: lambda bufs: quantize_int8(bufs["a"])})
