"""Layers of bfloat16 weights in a LinearStack, whose buffers are float16: the calls one by one into float16 outputs; a norm of another
type than the buffers is refused."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_bfloat16_layers_in_a_stack():
    from gemmlib_b200.int8_linear import Int8Linear, quantize_int8
    from gemmlib_b200.stack import LinearStack

    g = torch.Generator(device="cuda").manual_seed(0)
    w = [(torch.randn(64, 64, generator=g, device="cuda") * 0.1).bfloat16() for _ in range(2)]
    layers = [Int8Linear(w[0], torch.randn(64, generator=g, device="cuda").bfloat16()), Int8Linear(w[1])]
    stack = LinearStack([(layers[0], "x", "a"), (layers[1], "a", "b")])
    x = torch.randn(5, 64, generator=g, device="cuda").half()
    a = layers[0](quantize_int8(x), out=torch.empty(5, 64, dtype=torch.float16, device="cuda"))
    b = layers[1](quantize_int8(a), out=torch.empty_like(a))
    for given in (x, x.float()):
        got = stack.forward(given, "b")
        assert got.dtype == torch.float16 and torch.equal(got, b) and torch.equal(stack.buffers(5)["a"], a)


def test_a_bfloat16_norm_in_a_stack_is_refused():
    from gemmlib_b200.int8_linear import Int8Linear, RMSNormInt8
    from gemmlib_b200.stack import LinearStack

    norm = RMSNormInt8(torch.ones(64, device="cuda").bfloat16())
    stack = LinearStack([(Int8Linear(torch.ones(32, 64, device="cuda").half()), "x", "a")], int8_inputs={0: lambda bufs: norm(bufs["x"])})
    with pytest.raises(RuntimeError, match="one row of the input's length and type"):
        stack.forward(torch.ones(3, 64, device="cuda").half(), "a")
