"""Rows of the layer norm that leave no spread, or next to none beside their mean."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
WIDTHS = [1, 7, 64, 257, 300, 513, 1001, 2049, 4097, 8192, 8195, 12000, 16383, 16384]


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_a_row_of_equal_values_is_its_own_mean(blas, cols, dtype):
    """Whatever the value: the mean is that value to the last bit, nothing is left beside it, and y is b exactly."""
    g = torch.Generator().manual_seed(cols)
    value = torch.cat((torch.tensor([1000.1, 0.1, 333.337, -7.77, 1 / 3]), torch.rand(95, generator=g) * 1000 + 1)).to(dtype)
    x = value[:, None].expand(100, cols).contiguous().cuda()
    w, b = (torch.randn(cols, generator=g).cuda() for _ in range(2))
    y, mean, rstd = torch.empty_like(x), torch.empty(100, device="cuda"), torch.empty(100, device="cuda")
    blas.layer_norm(100, cols, x, w, b, 1e-5, y, mean, rstd)
    assert torch.equal(mean.cpu(), value.float())
    assert torch.equal(y, b.to(dtype).expand(100, cols))
    # 1 / sqrt(eps): eps itself, the root and the quotient are rounded
    assert torch.all((rstd.double() * 1e-5 ** 0.5 - 1).abs() <= 4 * U)


@pytest.mark.parametrize("cols", [300, 1001, 8192, 12000])
def test_rows_with_little_spread(blas, cols):
    """Values a few steps of FP32 around 1000: the mean is the nearest FP32 number or the next, so the deviations are off by
    at most one step of 2^-14 (512 <= x < 1024)."""
    g = torch.Generator().manual_seed(cols)
    step = 2.0 ** -14
    x = (1000 + torch.randint(-3, 4, (64, cols), generator=g).float() * step).cuda()
    y, mean, rstd = torch.empty_like(x), torch.empty(64, device="cuda"), torch.empty(64, device="cuda")
    blas.layer_norm(64, cols, x, None, None, 1e-5, y, mean, rstd)
    want = x.double().mean(1)
    assert torch.all((mean.double() - want).abs() <= step)
    # var is off by the mean's step squared at most, beside roundings
    var = ((x.double() - want[:, None]) ** 2).mean(1)
    r = 1 / torch.sqrt(var + 1e-5)
    assert torch.all((rstd.double() - r).abs() <= r * (40 * U + 0.5 * step ** 2 * r ** 2))


@pytest.mark.parametrize("cols", [5, 300, 1001, 8192, 16384])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_the_mean_of_a_row_with_an_infinity(blas, cols, dtype):
    """It is that infinity wherever it stands, NaN with two of different signs; nothing finite is left of the row."""
    x = torch.randn(6, cols, device="cuda").to(dtype)
    inf = float("inf")
    x[0, 0], x[1, cols // 2], x[2, cols - 1] = inf, -inf, inf
    x[3, 0], x[3, cols - 1] = inf, -inf
    x[4, cols // 3] = float("nan")
    y, mean, rstd = torch.empty_like(x), torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
    blas.layer_norm(6, cols, x, None, None, 1e-5, y, mean, rstd)
    assert mean[:3].tolist() == [inf, -inf, inf]
    assert torch.all(torch.isnan(mean[3:5])) and torch.all(torch.isnan(rstd[:5])) and torch.all(torch.isnan(y[:5]))
    assert torch.all(torch.isfinite(y[5])) and bool(torch.isfinite(mean[5]))
