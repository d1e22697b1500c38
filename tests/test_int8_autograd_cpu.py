"""The int8 operators have no derivatives: a tensor of a call that requires a gradient (while gradients are enabled) or has a
tangent is refused, before anything else is asked of it (so that no GPU is needed to see it)."""
import pytest

torch = pytest.importorskip("torch")


def x16():
    return torch.zeros(2, 32, dtype=torch.float16)


def rows(scales=None):
    from gemmlib_b200.int8_linear import Int8Rows

    return Int8Rows(torch.zeros(2, 32, dtype=torch.int8), torch.ones(2) if scales is None else scales)


def calls():
    """Each call with one tensor that the argument makes."""
    from gemmlib_b200.int8_linear import int8_linear, quantize_int8, rms_norm_int8, silu_mul_int8

    w = torch.ones(32, dtype=torch.float16)
    scales, out = torch.ones(2), torch.zeros(2, 2, dtype=torch.float16)
    return {
        "quantize": (x16(), quantize_int8),
        "norm": (x16(), lambda t: rms_norm_int8(t, w)),
        "norm's weight": (w, lambda t: rms_norm_int8(x16(), t)),
        "residual": (x16(), lambda t: rms_norm_int8(x16(), w, residual=t)),
        "residual_out": (x16(), lambda t: rms_norm_int8(x16(), w, residual=x16(), residual_out=t)),
        "gate": (x16(), lambda t: silu_mul_int8(t, x16())),
        "up": (x16(), lambda t: silu_mul_int8(x16(), t)),
        "dequantized scales": (scales, lambda t: rows(t).dequantize()),
        "scales": (scales, lambda t: int8_linear(rows(t), rows())),
        "weight's scales": (scales, lambda t: int8_linear(rows(), rows(t))),
        "bias": (out[0], lambda t: int8_linear(rows(), rows(), t)),
        "out": (out, lambda t: int8_linear(rows(), rows(), out=t)),
    }


NAMES = ["quantize", "norm", "norm's weight", "residual", "residual_out", "gate", "up", "dequantized scales", "scales",
         "weight's scales", "bias", "out"]


def test_every_call_is_named():
    assert list(calls()) == NAMES


@pytest.mark.parametrize("name", NAMES)
def test_a_tensor_that_requires_a_gradient_is_refused(name):
    tensor, call = calls()[name]
    with pytest.raises(RuntimeError, match="no backward pass"):
        call(tensor.clone().requires_grad_())
    with torch.no_grad(), pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        call(tensor.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        call(tensor)


def test_a_layer_of_given_rows_takes_their_scales_without_history():
    from gemmlib_b200.int8_linear import Int8Linear

    layer = Int8Linear.from_rows(rows(torch.ones(2, requires_grad=True) * 2))
    assert not layer.q_scales.requires_grad and layer.q_scales.tolist() == [2, 2]


@pytest.mark.parametrize("name", NAMES)
def test_a_tensor_with_a_tangent_is_refused(name):
    """Forward-mode derivatives, which no_grad does not turn off."""
    from torch.autograd import forward_ad

    tensor, call = calls()[name]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(tensor, torch.ones_like(tensor))
        with pytest.raises(RuntimeError, match="no forward derivatives"):
            call(dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no forward derivatives"):
            call(dual)
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call(forward_ad.unpack_dual(dual).primal)
