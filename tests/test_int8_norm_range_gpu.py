"""The norm of rows whose squares leave fp32 downwards, which an eps of nothing allows."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPS24 = 2.0 ** -24


@pytest.mark.parametrize("cols", [7, 300, 4096, 9000, 40000, 70000])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-38 * 1.18, 1e-5])
def test_a_scale_is_right_or_nan(cols, residual, eps):
    """fp32 sums as in the other tests of the norm: 47 roundings of 2^-24.  Below 2^-126 a sum is off by up to 2^-150 for every addition: of a
    mean of at least 2^-126 that is 2^-24 of it, halved by the root."""
    from gemmlib_b200.int8_linear import rms_norm_int8

    g = torch.Generator(device="cuda").manual_seed(cols)
    sizes = [1.0, 2.0 ** -30, 2.0 ** -61, 2.0 ** -66, 1e-25, 2.0 ** -120, 0.0]
    x = (torch.randn(len(sizes), cols, generator=g, device="cuda").double()
         * torch.tensor(sizes, dtype=torch.float64, device="cuda")[:, None]).to(torch.bfloat16)
    w = (1 + 0.1 * torch.randn(cols, generator=g, device="cuda")).bfloat16()
    rows = rms_norm_int8(x, w, eps, residual=torch.zeros_like(x))[0] if residual else rms_norm_int8(x, w, eps)
    e = float(torch.tensor(eps, dtype=torch.float32))
    t, mean = x.double() * w.double(), x.double().square().mean(1) + e
    want = t.abs().amax(1) / 127 / mean.sqrt()
    for i, size in enumerate(sizes):
        got = float(rows.scales[i])
        if size == 0.0:
            assert got == 0.0 and not rows.values[i].any()
        elif float(mean[i]) < 2.0 ** -126 * 0.99:
            assert got != got, (size, got)
        elif float(mean[i]) > 2.0 ** -126 * 1.01:
            # (a scale below 2^-126 is off by up to 2^-150)
            assert abs(got - float(want[i])) <= float(want[i]) * 48.5 * EPS24 + 2.0 ** -150, (size, got, float(want[i]))
