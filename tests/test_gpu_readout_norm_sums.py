"""Layer norm over many rows: sums of gradients that are alike, whose roundings are alike too."""
import pytest
import torch

from heliox_amd import readout

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24


@pytest.mark.parametrize("rows,width,dtype", [
    (3_000_000, 5, torch.float32), (500_000, 120, torch.float16), (400_001, 300, torch.float32), (300_000, 1100, torch.bfloat16),
    (100_000, 8192, torch.float16), (20_000, 12_000, torch.float32),    # held by the workgroups that make dx
    (20_001, 12_289, torch.float16), (20_000, 13_001, torch.float32), (6000, 131_073, torch.bfloat16), (3000, 300_000, torch.float32)])
def test_gradients_of_weight_and_bias(rows, width, dtype):
    """Every row and its gradient the same: the sums are `rows` times one term.  Up to 128 terms and 32 such sums, or
    those of 64 bits, are added one after another, each partial sum rounded: half of 160 halves of the sum, and three for a
    term and the result.  (Terms themselves: from the call's own mean and rstd.)"""
    gen = torch.Generator().manual_seed(width)
    x = torch.randn(1, width, generator=gen).to(dtype).cuda().expand(rows, width)
    dy = (0.5 + torch.rand(1, width, generator=gen)).to(dtype).cuda().expand(rows, width)
    _, mean, rstd = readout.layer_norm(x[:1])
    mean, rstd = mean.expand(rows).contiguous(), rstd.expand(rows).contiguous()
    _, dweight, dbias = readout.layer_norm_grad(x, None, mean, rstd, dy)
    torch.cuda.synchronize()
    n = (x[0].double() - mean[0].double()) * rstd[0].double()
    for got, term in ((dweight, dy[0].double() * n), (dbias, dy[0].double())):
        off = (got.double() - rows * term).abs() / (rows * term.abs()) / F32
        assert float(off.max()) <= 84, float(off.max())
    torch.cuda.empty_cache()
