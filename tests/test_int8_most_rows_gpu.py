"""As many rows as the C entry points' int holds: four a CTA, and 256 a CTA in the dequantization."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 200])
def test_rows_of_one_column(rows):
    from gemmlib_b200 import capi

    x = torch.full((rows,), 2.0, dtype=torch.float16, device="cuda")
    values = torch.zeros(rows, dtype=torch.int8, device="cuda")
    scales = torch.zeros(rows, device="cuda")
    x[-3:] = torch.tensor([-4.0, 0.0, 127.0])
    capi.int8_rows_quant(capi.INT8_FP16, rows, 1, (x, 1), (values, 1), scales)
    assert values[-3:].tolist() == [-127, 0, 127] and scales[-2:].tolist() == [0, 1]
    assert int(values[:-3].min()) == 127 and float(scales[:-3].min()) == float(scales[:-3].max()) == float(scales[0])
    out = torch.zeros(rows, dtype=torch.float16, device="cuda")
    capi.int8_rows_dequant(capi.INT8_FP16, rows, 1, (values, 1), scales, (out, 1))
    torch.cuda.synchronize()
    assert torch.equal(out, x)
