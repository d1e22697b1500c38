"""Layers of weights that are int8 already: whatever their layout, in memory of the layer's own."""
import pytest

torch = pytest.importorskip("torch")

LAYOUTS = {
    "rows of their own": lambda v: v.clone(),
    "columns of a wider matrix": lambda v: torch.cat([v[:, :3], v, v[:, :5]], 1)[:, 3: 3 + v.shape[1]],
    "columns on 16 bytes": lambda v: torch.cat([v[:, :16], v], 1)[:, 16:],
    "transposed": lambda v: v.t().contiguous().t(),
    "every second column": lambda v: v.repeat_interleave(2, 1)[:, ::2],
    "every second row": lambda v: v.repeat_interleave(2, 0)[::2],
}


def rows(n, k, device):
    g = torch.Generator().manual_seed(k)
    return (torch.randint(-127, 128, (n, k), generator=g).to(torch.int8).to(device),
            (torch.rand(n, generator=g) / 100).to(device))


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("k", [64, 63, 96])
def test_the_layers_weights_are_its_own_and_begin_on_32_bytes(layout, k):
    from gemmlib_b200.int8_linear import Int8Linear, Int8Rows

    values, scales = rows(40, k, "cpu")
    source = LAYOUTS[layout](values)
    layer = Int8Linear.from_rows(Int8Rows(source, scales))
    w = layer.q_weights
    assert w.is_contiguous() and w.shape[1] % 32 == 0 and w.shape[1] - k < 32
    assert torch.equal(w[:, :k], values) and not w[:, k:].any() and torch.equal(layer.q_scales, scales)
    want = values.clone(), scales.clone()
    source.zero_(), scales.zero_()
    assert torch.equal(w[:, :k], want[0]) and torch.equal(layer.q_scales, want[1])
    assert w.untyped_storage().data_ptr() != source.untyped_storage().data_ptr()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("k", [64, 63, 512])
@pytest.mark.parametrize("m", [1, 40])
def test_any_layout_gives_the_product_of_its_values(layout, k, m):
    from gemmlib_b200.int8_linear import Int8Linear, Int8Rows, int8_linear, quantize_int8

    values, scales = rows(48, k, "cuda")
    x = quantize_int8(torch.randn(m, k, device="cuda").half())
    padded = torch.zeros(48, -(-k // 32) * 32, dtype=torch.int8, device="cuda")
    padded[:, :k] = values
    want = int8_linear(x, Int8Rows(padded[:, :k], scales))
    source = LAYOUTS[layout](values)
    layer = Int8Linear.from_rows(Int8Rows(source, scales))
    assert torch.equal(layer(x), want)
    source.fill_(1), scales.fill_(1)
    for _ in range(2):  # the weights are fetched early now
        assert torch.equal(layer(x), want)
