"""Which products of one and two rows are streamed through registers: those that have a weight row (two rows: two) for each warp of the GPU at most, and no long
ones.  On the GPU, the tensor cores' results of the narrow and the short ones."""
import pytest

torch = pytest.importorskip("torch")

# rows, in_features, out_features
STREAMED = [(1, 1024, 1024), (1, 1408, 2048), (1, 4096, 3552), (1, 64, 3552), (1, 1, 1), (2, 1024, 2048), (2, 512, 4700), (2, 2560, 512), (2, 2816, 2048)]
MULTIPLIED = [(1, 512, 12000), (1, 200, 28672), (1, 28672, 200), (1, 8192, 512), (1, 16384, 300), (1, 512, 8192), (1, 64, 20000), (1, 4096, 4096),
              (2, 8192, 512), (2, 512, 8192), (2, 4096, 512), (2, 64, 28672), (2, 300, 16384), (3, 64, 64)]


def test_choices(lib_built):
    from gemmlib_b200 import capi

    for m, k, n in STREAMED:
        assert capi.fp8_gemm_plan(m, n, k)["kernel"] == "stream", (m, k, n)
    for m, k, n in MULTIPLIED:
        assert capi.fp8_gemm_plan(m, n, k)["kernel"] == "few", (m, k, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", STREAMED + MULTIPLIED + [(1, 17, 3552), (2, 2800, 2239), (2, 15, 4736), (1, 33, 3553), (2, 30, 4737)],
                         ids=lambda s: "x".join(map(str, s)))
def test_products(shape, dtype):
    from gemmlib_b200 import ms_blkq4linear_ext as ext
    from gemmlib_b200.fp8_linear import fp8_linear
    from tests.test_fp8_linear_gpu import check_close, rows_of, weight_of

    m, k, n = shape
    x, w = rows_of(m, k, 1), weight_of(n, k, 2)
    bias = torch.linspace(-3, 3, n, device="cuda").to(dtype)
    out = fp8_linear(x, w, bias, dtype=dtype)
    check_close(out, x, w, bias)
    assert torch.equal(fp8_linear(x, w, bias, dtype=dtype, flags=ext.EARLY_WEIGHT_FETCH), out)
