"""Layer norm's gradient of rows whose mean, times 1 / deviation, is more than a float holds: (x - mean) / deviation is finite in
every column, and the gradient is too."""
import pytest
import torch

from hetuctr_amd import nn
from tests import dense_reference64 as ref64

gpu = pytest.mark.gpu
WIDTHS = [1, 2, 3, 4, 5, 6, 7, 8, 9, 15, 17, 20, 37, 64, 100, 130, 200, 333, 520, 600, 601, 1000, 1100, 1443, 2500, 4100, 4101, 5000, 9000, 9001,
          16384, 16388]


@gpu
@pytest.mark.parametrize("stream, act", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("width", WIDTHS)
def test_gradient_of_rows_far_from_zero_is_finite(width, stream, act, add):
    # rows that hold 2^126 everywhere: no deviation, and 1 / sqrt(eps) in its place
    rows = 1030
    level = torch.tensor(2.0 ** 126, device="cuda", dtype=stream)
    x = level.expand(rows, width).clone()
    mean, rstd = torch.full((rows,), 2.0 ** 126, device="cuda"), torch.full((rows,), 1e-5 ** -0.5, device="cuda")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(width)
    dy = torch.randn((rows, width), device="cuda", generator=gen).to(act)
    weight = torch.full((width,), 1.5, device="cuda")
    if add:
        dx, dresidual, dweight, dbias = nn.dropout_add_layer_norm_backward(dy, None, x, mean, rstd, weight, weight)
    else:
        dx, dweight, dbias = nn.layer_norm_backward(dy, x, mean, rstd, weight, weight)
    # x - mean is 0 everywhere: dx = rstd * (g - its mean), dweight = 0
    (want, _, sums), (size, _, total) = ref64.gradient(dy.double(), torch.zeros_like(x, dtype=torch.float64), torch.zeros((rows, 1), device="cuda"),
                                                       rstd.double()[:, None], weight.double())
    assert torch.isfinite(dx).all()
    # a sum of `width` values, in 20 terms of a lane and pairs at most, and a rounding to the type: 64 units and 2^-8 or 2^-24
    unit = 2.0 ** -8 if dx.dtype == torch.bfloat16 else 2.0 ** -24
    assert ((dx.double() - want).abs() <= 64 * 2.0 ** -24 * size + unit * want.abs() + 2.0 ** -126).all()
    assert (dweight == 0).all()
    assert ((dbias.double() - sums).abs() <= (300 * 2.0 ** -24) * total).all()
