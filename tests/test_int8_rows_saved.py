"""Int8Rows through torch.save, pickle, copy and another process' queue: the operators' values and scales share one storage, which
torch.save refuses of tensors of two types."""
import copy
import io
import pickle

import pytest

torch = pytest.importorskip("torch")


def shared(n, k, device):
    """Rows as the operators lay them out: on 32 bytes, the scales behind them."""
    from gemmlib_b200.int8_linear import Int8Rows

    pitch = -(-k // 32) * 32
    both = torch.zeros(n * (pitch + 4), dtype=torch.int8, device=device)
    g = torch.Generator().manual_seed(0)
    values, scales = both[:n * pitch].view(n, pitch)[:, :k], both[n * pitch:].view(torch.float32)
    values.copy_(torch.randint(-127, 128, (n, k), generator=g))
    scales.copy_(torch.rand(n, generator=g))
    return Int8Rows(values, scales)


def saved(x):
    file = io.BytesIO()
    torch.save(x, file)
    file.seek(0)
    return torch.load(file)


WAYS = {"save": saved, "pickle": lambda x: pickle.loads(pickle.dumps(x)), "deepcopy": copy.deepcopy, "copy": copy.copy,
        "in a dict": lambda x: saved({"layer": [x, 1]})["layer"][0]}


def check(rows, back):
    from gemmlib_b200.int8_linear import Int8Rows

    assert type(back) is Int8Rows and back.values.dtype == torch.int8 and back.scales.dtype == torch.float32
    assert torch.equal(back.values, rows.values) and torch.equal(back.scales, rows.scales)
    assert back.values.device == rows.values.device and back.scales.device == rows.scales.device


@pytest.mark.parametrize("way", list(WAYS))
@pytest.mark.parametrize("n,k", [(5, 64), (3, 33), (1, 1)])
def test_rows_come_back(way, n, k):
    rows = shared(n, k, "cpu")
    check(rows, WAYS[way](rows))


@pytest.mark.gpu
@pytest.mark.parametrize("way", list(WAYS))
def test_rows_of_an_operator_come_back(way):
    from gemmlib_b200.int8_linear import Int8Linear, int8_linear, quantize_int8

    rows = quantize_int8(torch.randn(40, 100, device="cuda").half())
    back = WAYS[way](rows)
    check(rows, back)
    assert torch.equal(back.dequantize(), rows.dequantize())
    x = quantize_int8(torch.randn(3, 100, device="cuda").half())
    assert torch.equal(Int8Linear.from_rows(back)(x), int8_linear(x, rows))
