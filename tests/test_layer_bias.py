"""The bias of the 8-bit layers is part of them: of their state, of a move, of a copy."""
import copy
import io

import pytest

torch = pytest.importorskip("torch")
E4M3 = torch.float8_e4m3fn


def fp8(bias, n=130, k=64, device="cpu"):
    from gemmlib_b200.fp8_linear import Fp8Linear, Fp8Weight

    w = torch.full((n, k), 2.0, device=device).to(E4M3)
    return Fp8Linear.from_weight(Fp8Weight(w, torch.ones(-(-n // 128), 1, device=device)), bias, torch.float16)


def int8(bias, n=130, k=64, device="cpu"):
    from gemmlib_b200.int8_linear import Int8Linear, Int8Rows

    return Int8Linear.from_rows(Int8Rows(torch.full((n, k), 2, dtype=torch.int8, device=device), torch.ones(n, device=device)), bias)


LAYERS = {"fp8": fp8, "int8": int8}


def ramp(n=130, device="cpu"):
    return torch.linspace(-3, 3, n, device=device).half()


@pytest.mark.parametrize("kind", LAYERS)
def test_the_state_has_the_bias(kind):
    make = LAYERS[kind]
    layer, other = make(ramp()), make(torch.zeros(130, dtype=torch.float16))
    held = io.BytesIO()
    torch.save(layer.state_dict(), held)
    held.seek(0)
    other.load_state_dict(torch.load(held))
    assert torch.equal(other.bias, ramp()) and "bias" not in make(None).state_dict() and make(None).bias is None
    with pytest.raises(RuntimeError, match="bias"):  # neither dropped nor made up
        make(None).load_state_dict(layer.state_dict())
    with pytest.raises(RuntimeError, match="bias"):
        layer.load_state_dict(make(None).state_dict())


@pytest.mark.parametrize("kind", LAYERS)
def test_states_that_were_saved_without_it_are_loaded(kind):
    make = LAYERS[kind]
    layer, old = torch.nn.Sequential(make(ramp()), make(None)), torch.nn.Sequential(make(None), make(None)).state_dict()
    for m in old._metadata.values():
        m["version"] = 1
    for state in (old, dict(old)):
        layer.load_state_dict(state)
        assert torch.equal(layer[0].bias, ramp()) and "0.bias" not in state


@pytest.mark.parametrize("kind", LAYERS)
def test_the_bias_moves_and_is_copied(kind):
    make = LAYERS[kind]
    given = ramp()
    layer = make(given)
    given.zero_()  # the layer of given weights has a copy of it
    assert torch.equal(layer.bias, ramp()) and torch.equal(copy.deepcopy(layer).bias, ramp())
    converted = copy.deepcopy(layer).bfloat16().bias
    assert converted.dtype == torch.float16 and torch.equal(converted, ramp())
    assert layer.to("meta").bias.device.type == "meta"
    given = torch.nn.Parameter(ramp())
    kept = make(given).bias
    assert isinstance(kept, torch.nn.Parameter) and kept is not given and kept.requires_grad and torch.equal(kept, ramp())
    assert make(ramp().requires_grad_()).bias.requires_grad  # which a call refuses while gradients are enabled


@pytest.mark.parametrize("kind", LAYERS)
def test_a_state_is_not_loaded_into_what_was_given(kind):
    make = LAYERS[kind]
    given = torch.zeros(130, dtype=torch.float16)
    layer, other = make(given), make(given)
    layer.load_state_dict(make(ramp()).state_dict())
    assert torch.equal(layer.bias, ramp()) and not given.any() and not other.bias.any()


@pytest.mark.parametrize("kind", LAYERS)
def test_layers_that_were_pickled_with_a_plain_attribute(kind):
    for bias in (ramp(), None):
        old = LAYERS[kind](bias)
        old.__dict__["bias"] = old._buffers.pop("bias")
        held = io.BytesIO()
        torch.save(old, held)
        held.seek(0)
        layer = torch.load(held, weights_only=False)
        assert "bias" not in layer.__dict__ and "bias" in layer._buffers and (layer.bias is None if bias is None else torch.equal(layer.bias, bias))
        assert ("bias" in layer.state_dict()) == (bias is not None) and layer.to("meta") is layer


@pytest.mark.gpu
@pytest.mark.parametrize("kind", LAYERS)
def test_restored_and_moved_layers_on_the_gpu(kind):
    make = LAYERS[kind]
    layer = make(ramp(device="cuda"), device="cuda")
    x = torch.randn(5, 64, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").half()
    want = layer(x)
    assert not torch.equal(want, make(None, device="cuda")(x))
    other = make(torch.zeros(130, dtype=torch.float16, device="cuda"), device="cuda")
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), want)
    for moved in (make(ramp()).cuda(), copy.deepcopy(layer).cpu().cuda()):  # the first one was made without a GPU
        assert torch.equal(moved(x), want) and moved.bias.is_cuda


@pytest.mark.gpu
def test_layers_that_quantize_keep_a_parameter_as_one():
    from gemmlib_b200.fp8_linear import Fp8Linear
    from gemmlib_b200.int8_linear import Int8Linear

    plain = torch.nn.Linear(64, 130, device="cuda", dtype=torch.float16)
    for cls in (Fp8Linear, Int8Linear):
        layer = cls(plain.weight, plain.bias)
        assert layer.bias is plain.bias and "bias" in layer.state_dict()
        given = plain.bias.detach()
        layer = cls(plain.weight, given)
        assert "bias" in dict(layer.named_buffers()) and layer.bias.data_ptr() != given.data_ptr() and torch.equal(layer.bias, given)
        with torch.no_grad():
            assert torch.equal(layer(torch.zeros(2, 64, device="cuda").half())[1], given)
        assert layer.double().bias.dtype == torch.float16
