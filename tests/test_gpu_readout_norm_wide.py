"""Layer norm of rows far wider than registers hold, whose values are alike: so are the roundings of their sums."""
import pytest
import torch

from heliox_amd import readout
from readout_util import UNIT

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24


@pytest.mark.parametrize("width", [32_769, 1 << 20, (1 << 22) + 1, 1 << 24])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("size", [0.7, 1.3, 0.9])
def test_rows_of_two_values(width, dtype, size):
    """+-size in turns about 0.25, g of three values: at most 8 terms are added in fp32, 7 halves of a step, the sums of
    these in 64 bits, those of 64 lanes and 16 waves in fp32, of partial sums half of 6 + 16.  rstd takes half of the
    variance's 18 + 4, 1 / sqrt 3 more, n and y four."""
    sign = 1 - 2 * (torch.arange(width, device="cuda") % 2)
    x = torch.stack([(0.25 + size * sign), (0.25 - size * sign)]).to(dtype)
    dy = torch.stack([0.5 + 0.3 * (torch.arange(width, device="cuda") % 3), 0.6 + 0.1 * (torch.arange(width, device="cuda") % 5)]).to(dtype)
    wide, g = x.double(), dy.double()
    mean = wide.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((wide - mean) ** 2).mean(1, keepdim=True) + 1e-5)
    n = (wide - mean) * rstd
    dx = rstd * (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True))
    y, got_mean, got_rstd = readout.layer_norm(x)
    got_dx = readout.layer_norm_grad(x, None, got_mean, got_rstd, dy, parameters=False)[0]
    torch.cuda.synchronize()
    unit = UNIT[dtype]
    assert float((got_mean[:, None].double() - mean).abs().max()) <= 20 * F32 * (size + 0.25)
    assert float((got_rstd[:, None].double() / rstd - 1).abs().max()) <= 16 * F32
    assert bool(((y.double() - n).abs() <= (unit + 20 * F32) * n.abs() + 20 * F32).all())
    # g, its mean and n times the mean of g n, which n's own error reaches too; all of them at most 1.1
    assert bool(((got_dx.double() - dx).abs() <= unit * dx.abs() + 64 * F32 * rstd * 1.1 + 2.0 ** -25).all())
    torch.cuda.empty_cache()
