"""Writes of the int8 operators into a caller's tensor are seen by autograd, which may have saved it."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def writers():
    from gemmlib_b200.int8_linear import int8_linear, quantize_int8, rms_norm_int8

    w = torch.randn(48, 32, device="cuda").half()
    x, rows, weight = torch.randn(4, 48, device="cuda").half(), quantize_int8(w), torch.ones(48, device="cuda").half()
    residual = torch.randn(4, 48, device="cuda").half()
    return {
        "sum in a tensor of its own": lambda t: rms_norm_int8(x, weight, residual=residual, residual_out=t),
        "sum over the input": lambda t: rms_norm_int8(t, weight, residual=residual, residual_out=t),
        "sum over the residual": lambda t: rms_norm_int8(x, weight, residual=t, residual_out=t),
        "product": lambda t: int8_linear(quantize_int8(w[:4]), rows, out=t),
    }


NAMES = ["sum in a tensor of its own", "sum over the input", "sum over the residual", "product"]


@pytest.mark.parametrize("name", NAMES)
def test_a_saved_tensor_that_is_written_is_noticed(name):
    write = writers()[name]
    factor = torch.ones(4, 48, dtype=torch.float16, device="cuda", requires_grad=True)
    for view in (lambda t: t, lambda t: t[:, :48], lambda t: t.view(2, 2, 48).view(4, 48)):
        saved = torch.randn(4, 48, device="cuda").half()
        y = (factor * saved).sum()  # keeps `saved` for the gradient of `factor`
        before = saved._version
        write(view(saved))
        assert saved._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


@pytest.mark.parametrize("name", NAMES)
def test_what_is_only_read_keeps_its_version_and_inference_tensors_are_written(name):
    from gemmlib_b200.int8_linear import int8_linear, quantize_int8, rms_norm_int8, silu_mul_int8

    write = writers()[name]
    with torch.inference_mode():
        made = torch.zeros(4, 48, dtype=torch.float16, device="cuda")
        write(made)
    write(made)
    assert made.any()
    x, w = torch.randn(4, 48, device="cuda").half(), torch.ones(48, device="cuda").half()
    rows = quantize_int8(x)
    rms_norm_int8(x, w), rms_norm_int8(x, w, residual=x), silu_mul_int8(x, x), rows.dequantize(), int8_linear(rows, rows)
    assert [t._version for t in (x, w, *rows)] == [0] * 4
