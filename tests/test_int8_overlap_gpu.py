"""Outputs of the int8 operators in a caller's memory: refused where they overlap what the call reads, taken where they lie beside it."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

M, N, K = 24, 32, 64


def operands(slab):
    """Rows, weights, their scales and a bias, each in 4 KB of `slab` (bytes) of its own; views that end where the next begins."""
    from gemmlib_b200.int8_linear import Int8Rows

    g = torch.Generator(device="cuda").manual_seed(0)
    at = lambda i, n: slab[4096 * i + 4096 - n: 4096 * i + 4096]
    x, w = at(0, M * K).view(torch.int8).view(M, K), at(1, N * K).view(torch.int8).view(N, K)
    xs, ws, bias = at(2, 4 * M).view(torch.float32), at(3, 4 * N).view(torch.float32), at(4, 2 * N).view(torch.float16)
    x.copy_(torch.randint(-128, 128, x.shape, generator=g, device="cuda"))
    w.copy_(torch.randint(-128, 128, w.shape, generator=g, device="cuda"))
    xs.copy_(torch.rand(M, generator=g, device="cuda") / 100)
    ws.copy_(torch.rand(N, generator=g, device="cuda") / 10)
    bias.copy_(torch.randn(N, generator=g, device="cuda"))
    return Int8Rows(x, xs), Int8Rows(w, ws), bias


@pytest.mark.parametrize("of", ["rows", "weights", "scales", "weights' scales", "bias"])
@pytest.mark.parametrize("pitch", [N, 2 * N])
def test_a_product_into_its_operands_is_refused(of, pitch):
    from gemmlib_b200.int8_linear import int8_linear

    slab = torch.zeros(10 * 4096, dtype=torch.uint8, device="cuda")
    x, w, bias = operands(slab)
    want = int8_linear(x, w, bias)
    end = 4096 * (1 + ["rows", "weights", "scales", "weights' scales", "bias"].index(of))
    begin = end - {"rows": M * K, "weights": N * K, "scales": 4 * M, "weights' scales": 4 * N, "bias": 2 * N}[of]
    size = 2 * ((M - 1) * pitch + N)

    def out(first_byte):
        return slab[first_byte: first_byte + size].view(torch.float16).as_strided((M, N), (pitch, 1))

    before = slab.clone()
    for first in (end - 16, begin - size + 16):  # its last bytes, its first ones
        with pytest.raises(RuntimeError, match="out overlaps a tensor"):
            int8_linear(x, w, bias, out=out(first + (-first % 2)) if first >= 0 else out(end - 2))
    assert torch.equal(slab, before)
    assert torch.equal(int8_linear(x, w, bias, out=out(5 * 4096)), want)  # right behind the bias


def test_operands_and_output_as_columns_of_one_matrix():
    """Bytes of one pitch, none shared: every tensor of the call in columns of its own, or rows."""
    from gemmlib_b200.int8_linear import Int8Rows, int8_linear

    slab = torch.zeros(10 * 4096, dtype=torch.uint8, device="cuda")
    x, w, bias = operands(slab)
    want = int8_linear(x, w, bias)
    wide = torch.zeros(40, 320, dtype=torch.uint8, device="cuda")
    rows, weights = wide[:M, 64: 64 + K].view(torch.int8), wide[:N, 128: 128 + K].view(torch.int8)
    rows.copy_(x.values), weights.copy_(w.values)
    xs, b = wide[39, :4 * M].view(torch.float32), wide[38, 192: 192 + 2 * N].view(torch.float16)
    xs.copy_(x.scales), b.copy_(bias)
    out = wide[:, 192: 192 + 2 * N].view(torch.float16)
    keep = wide.clone()
    assert torch.equal(int8_linear(Int8Rows(rows, xs), Int8Rows(weights, w.scales), b, out=out[:M]), want)
    keep[:M, 192: 192 + 2 * N] = want.view(torch.uint8)
    assert torch.equal(wide, keep)
    for bad in (out[39 - M: 39], wide[:M, 190: 190 + 2 * N].view(torch.float16), wide[1: M + 1, 126: 126 + 2 * N].view(torch.float16)):
        with pytest.raises(RuntimeError, match="out overlaps a tensor"):  # the row of the bias, columns of the weights
            int8_linear(Int8Rows(rows, xs), Int8Rows(weights, w.scales), b, out=bad)


def test_a_sum_beside_the_norms_weight():
    from gemmlib_b200.int8_linear import rms_norm_int8

    wide = torch.randn(6, 128, device="cuda").half()
    x, r, weight = torch.randn(4, 64, device="cuda").half(), torch.randn(4, 64, device="cuda").half(), wide[2, 64:]
    want, h = rms_norm_int8(x, weight.clone(), residual=r)
    got, same = rms_norm_int8(x, weight, residual=r, residual_out=wide[:4, :64])
    assert torch.equal(got.values, want.values) and torch.equal(got.scales, want.scales) and torch.equal(same, h)
    with pytest.raises(RuntimeError, match="overlaps the weight"):
        rms_norm_int8(x, weight, residual=r, residual_out=wide[:4, 1:65])
