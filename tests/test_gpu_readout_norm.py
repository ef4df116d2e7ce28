"""Layer norm and its gradient on the GPU against the formulas in 64 bits."""
import pytest
import torch

from heliox_amd import HelioxError, readout
from readout_util import UNIT, captured

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
F32 = 2.0 ** -24
# Every way a row is held, and its borders: single elements, whole and broken pieces of 4 or 8,
# 8 to 1024 lanes of one to four pieces, rows that are read again.
WIDTHS = [1, 2, 3, 4, 7, 8, 9, 31, 64, 65, 129, 257, 500, 512, 1000, 1001, 1024, 2047, 2048, 2049, 4096, 5000, 8192,
          8193, 16384, 16389, 32768, 32769, 40001]


def formulas(x, weight, bias, dy, eps=1e-5):
    x, dy = x.detach().cpu().double(), dy.detach().cpu().double()
    weight = torch.ones(x.shape[-1], dtype=torch.float64) if weight is None else weight.cpu().double()
    bias = torch.zeros(x.shape[-1], dtype=torch.float64) if bias is None else bias.cpu().double()
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    n = (x - mean) * rstd
    g = dy * weight
    dx = rstd * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    columns = lambda t: t.reshape(-1, x.shape[-1]).sum(0)  # noqa: E731
    return dict(y=n * weight + bias, mean=mean[..., 0], rstd=rstd[..., 0], dx=dx, dweight=columns(dy * n),
                dbias=columns(dy), n=n, g=g, off=x.abs().mean(-1, keepdim=True) * rstd)


def check(x, weight, bias, dy, eps=1e-5):
    """Errors against what sums of fp32 may be off by.  A sum over a row adds at most 32 values one
    after another and joins the rest in at most 10 steps, so a mean is off by at most 48 halves of
    a step of the mean size; `off` is that size in units of the row's own.  What follows takes
    fewer than 16 further operations.  A column's sum adds its rows one after another, in at most
    512 runs, then 32 runs after another and 16 of those."""
    want = formulas(x, weight, bias, dy, eps)
    y, mean, rstd = readout.layer_norm(x, weight, bias, eps=eps)
    dx, dweight, dbias = readout.layer_norm_grad(x, weight, mean, rstd, dy)
    torch.cuda.synchronize()
    assert y.dtype == dx.dtype == x.dtype and mean.dtype == rstd.dtype == dweight.dtype == dbias.dtype == torch.float32
    got = {k: v.cpu().double() for k, v in dict(y=y, mean=mean, rstd=rstd, dx=dx, dweight=dweight, dbias=dbias).items()}
    unit = UNIT[x.dtype]
    loose = 64 * F32 * (1 + want["off"])                       # of n, in its own units
    w = torch.ones(x.shape[-1]) if weight is None else weight.cpu()
    near = unit * want["y"].abs() + loose * (1 + want["n"].abs()) * w.double().abs() + 4 * F32 * want["y"].abs()
    if x.dtype == torch.float16:
        near += 2.0 ** -25
    assert bool(((got["y"] - want["y"]).abs() <= near).all())
    assert bool(((got["mean"] - want["mean"]).abs() <= 48 * F32 * x.cpu().double().abs().mean(-1)).all())
    assert bool(((got["rstd"] / want["rstd"] - 1).abs() <= 64 * F32 * (1 + want["off"][..., 0])).all())
    # (g - mean g) - n mean(g n): each term off by its own sums
    size = want["rstd"][..., None] * (want["g"].abs() + want["g"].abs().mean(-1, keepdim=True)
                                      + (1 + want["n"].abs()) * (want["g"] * want["n"]).abs().mean(-1, keepdim=True))
    near = unit * want["dx"].abs() + 4 * loose * size
    if x.dtype == torch.float16:
        near += 2.0 ** -25
    assert bool(((got["dx"] - want["dx"]).abs() <= near).all())
    columns = lambda t: t.reshape(-1, x.shape[-1]).sum(0)  # noqa: E731
    rows = max(1, x.numel() // x.shape[-1])
    chain = -(-rows // min(rows, 64)) + 32 + 16 + 8
    dy_, n = dy.cpu().double().abs(), want["n"].abs()
    assert bool(((got["dweight"] - want["dweight"]).abs() <= columns(dy_ * (n * chain * F32 + loose * (1 + n)))).all())
    assert bool(((got["dbias"] - want["dbias"]).abs() <= columns(dy_ * chain * F32)).all())


def normal(seed, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale + shift).to(dtype).cuda()


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", TYPES)
def test_widths(width, dtype):
    rows = 37 if width < 5000 else 5
    check(normal(0, rows, width, dtype=dtype, scale=2.0, shift=0.5), normal(1, width, shift=1.0), normal(2, width),
          normal(3, rows, width, dtype=dtype))


@pytest.mark.parametrize("rows", [1, 2, 31, 32, 33, 515, 2600])
@pytest.mark.parametrize("width,dtype", [(5, torch.float32), (24, torch.bfloat16), (120, torch.float16),
                                         (601, torch.float32), (3001, torch.bfloat16)])
def test_rows(rows, width, dtype):
    """Fewer rows than a workgroup takes, and more than the workgroups take at once."""
    check(normal(0, rows, width, dtype=dtype), normal(1, width, shift=1.0), normal(2, width),
          normal(3, rows, width, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", TYPES)
def test_types_of_the_weights(dtype, kind):
    check(normal(0, 9, 100, dtype=dtype), normal(1, 100, dtype=kind, shift=1.0), normal(2, 100, dtype=kind),
          normal(3, 9, 100, dtype=dtype))


@pytest.mark.parametrize("weight,bias", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("width", [3, 130, 40001])
def test_without_weight_or_bias(weight, bias, width):
    check(normal(0, 6, width), normal(1, width) if weight else None, normal(2, width) if bias else None, normal(3, 6, width))


def test_voltages_far_from_zero():
    """Captured voltages: the mean is many times their spread, and the variance no difference of squares."""
    x = normal(0, 20, 500, scale=0.01, shift=-65.0)
    check(x, normal(1, 500, shift=1.0), normal(2, 500), normal(3, 20, 500))


@pytest.mark.parametrize("width", [60, 500, 3000, 40001])
def test_a_mean_far_from_zero_keeps_its_bits(width):
    """Rows at -65 of spread 8: the mean is off by what its own corrected sum is, not by what the sum of the
    values is: half a step of 65 and a few of the spread, in all 8 halves of a step of either."""
    x = normal(0, 40, width, scale=8.0, shift=-65.0)
    y, mean, _ = readout.layer_norm(x)
    want = formulas(x, None, None, x)
    assert bool(((mean.cpu().double() - want["mean"]).abs() <= F32 * 65 * 1.5 + 8 * F32 * 8).all())
    assert float((y.cpu().double() - want["y"]).norm()) <= 4 * F32 * float(want["y"].norm())


def test_views_and_shapes():
    wide = normal(0, 5, 7, 260, dtype=torch.bfloat16)
    x = wide[..., 3:103]                                       # rows that start at odd addresses
    dy = normal(3, 5, 7, 100, dtype=torch.bfloat16)
    check(x, normal(1, 100), normal(2, 100), dy)
    check(x.transpose(0, 1), normal(1, 100), normal(2, 100), dy.transpose(0, 1))
    check(wide[0, 0, ::2], normal(1, 130), normal(2, 130), normal(4, 130, dtype=torch.bfloat16))   # one row, not contiguous
    check(normal(5, 1, 100).expand(9, 100), normal(1, 100), normal(2, 100), normal(6, 1, 100).expand(9, 100))


def test_nothing_to_do():
    x = torch.empty(0, 4, 10, device="cuda")
    y, mean, rstd = readout.layer_norm(x)
    assert y.shape == x.shape and mean.shape == rstd.shape == (0, 4)
    dx, dweight, dbias = readout.layer_norm_grad(x, None, mean, rstd, x)
    assert dx.shape == x.shape and bool((dweight == 0).all()) and bool((dbias == 0).all())


def test_without_parameters():
    x, w, dy = normal(0, 11, 70), normal(1, 70), normal(2, 11, 70)
    _, mean, rstd = readout.layer_norm(x, w)
    whole = readout.layer_norm_grad(x, w, mean, rstd, dy)
    alone = readout.layer_norm_grad(x, w, mean, rstd, dy, parameters=False)
    assert torch.equal(whole[0], alone[0]) and alone[1] is None and alone[2] is None


@pytest.mark.parametrize("width", [6, 300, 40001])
def test_what_is_not_finite_stays_in_its_row(width):
    x, w, b, dy = normal(0, 40, width), normal(1, width), normal(2, width), normal(3, 40, width)
    y, mean, rstd = readout.layer_norm(x, w, b)
    dx = readout.layer_norm_grad(x, w, mean, rstd, dy)[0]
    x[7, 1], x[30, 0] = float("nan"), float("inf")
    y2, mean2, rstd2 = readout.layer_norm(x, w, b)
    dx2 = readout.layer_norm_grad(x, w, mean2, rstd2, dy)[0]
    keep = torch.ones(40, dtype=torch.bool)
    keep[7] = keep[30] = False
    assert torch.equal(y[keep], y2[keep]) and torch.equal(dx[keep], dx2[keep])
    assert bool(y2[~keep].isnan().any(1).all()) and bool(dx2[~keep].isnan().any(1).all())


def test_rows_of_one_value():
    """No spread: the output is the bias, the gradient by x g - mean(g) times 1 / sqrt(eps)."""
    x = torch.full((3, 64), 5.0, device="cuda")
    w, b, dy = normal(1, 64), normal(2, 64), normal(3, 3, 64)
    check(x, w, b, dy)
    assert torch.equal(readout.layer_norm(x, w, b)[0], b.expand(3, 64))


def test_gradients_against_differences():
    """Central differences of a smooth function in 64 bits, around the kernel's own inputs: the
    kernel's gradient is fp32, the differences' error of second order 1e-8 of it."""
    x, w, b, dy = normal(0, 4, 33), normal(1, 33, shift=1.0), normal(2, 33), normal(3, 4, 33)
    _, mean, rstd = readout.layer_norm(x, w, b)
    got = readout.layer_norm_grad(x, w, mean, rstd, dy)
    loss = lambda x, w, b: float((formulas(x, w, b, dy)["y"] * dy.cpu().double()).sum())  # noqa: E731
    for which, grad in enumerate(got):
        args = [x.cpu().double(), w.cpu().double(), b.cpu().double()]
        way = torch.randn(grad.shape, generator=torch.Generator().manual_seed(9), dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            moved = list(args)
            moved[which] = args[which] + sign * 1e-4 * way
            ends.append(loss(*moved))
        slope = float((grad.cpu().double() * way).sum())
        assert abs((ends[0] - ends[1]) / 2e-4 - slope) <= 1e-5 * float(grad.cpu().double().norm() * way.norm())


@pytest.mark.parametrize("width", [40, 3000, 40001])
def test_captured(width):
    x, w, b, dy = normal(0, 70, width), normal(1, width), normal(2, width), normal(3, 70, width)

    def call():
        y, mean, rstd = readout.layer_norm(x, w, b)
        return [y, mean, rstd, *readout.layer_norm_grad(x, w, mean, rstd, dy)]

    captured(call, lambda gen: (x.copy_(torch.randn(70, width, generator=gen)), dy.copy_(torch.randn(70, width, generator=gen))))


def test_streams_of_their_own():
    x, w = normal(0, 300, 1000), normal(1, 1000)
    want = readout.layer_norm(x, w)[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(readout.layer_norm(x, w)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(want, g) for g in got)


def test_in_an_autograd_function():
    class Norm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w, b):
            y, mean, rstd = readout.layer_norm(x, w, b)
            ctx.save_for_backward(x, w, mean, rstd)
            return y

        @staticmethod
        def backward(ctx, dy):
            x, w, mean, rstd = ctx.saved_tensors
            return readout.layer_norm_grad(x, w, mean, rstd, dy)

    x, w, b, dy = normal(0, 5, 50), normal(1, 50), normal(2, 50), normal(3, 5, 50)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    Norm.apply(*leaves).backward(dy)
    with torch.no_grad():
        _, mean, rstd = readout.layer_norm(x, w, b)
        want = readout.layer_norm_grad(x, w, mean, rstd, dy)
    assert all(torch.equal(leaf.grad, g) for leaf, g in zip(leaves, want))


def test_refusals():
    x, w = normal(0, 4, 6), normal(1, 6)
    _, mean, rstd = readout.layer_norm(x, w)
    for call, error, text in (
            (lambda: readout.layer_norm(x, w[:5]), ValueError, "weight has shape"),
            (lambda: readout.layer_norm(x, w, w.half()), TypeError, "bias is"),
            (lambda: readout.layer_norm(x, w.double()), TypeError, "not float32"),
            (lambda: readout.layer_norm(x.double()), TypeError, "not float32"),
            (lambda: readout.layer_norm(x, w.cpu()), ValueError, "GPU"),
            (lambda: readout.layer_norm(x, [1.0]), TypeError, "tensor"),
            (lambda: readout.layer_norm(x[0, 0]), ValueError, "width"),
            (lambda: readout.layer_norm(x[:, :0]), ValueError, "width"),
            (lambda: readout.layer_norm(x, eps=-1.0), HelioxError, "eps"),
            (lambda: readout.layer_norm(x, eps=float("nan")), HelioxError, "eps"),
            (lambda: readout.layer_norm(x, eps="1"), TypeError, "eps"),
            (lambda: readout.layer_norm(x.clone().requires_grad_()), ValueError, "records no graph"),
            (lambda: readout.layer_norm_grad(x, w, mean, rstd, x[:3]), ValueError, "dy has shape"),
            (lambda: readout.layer_norm_grad(x, w, mean, rstd, x.half()), TypeError, "dy is"),
            (lambda: readout.layer_norm_grad(x, w, mean[:3], rstd, x), ValueError, "mean has shape"),
            (lambda: readout.layer_norm_grad(x, w, mean, None, x), TypeError, "rstd"),
            (lambda: readout.layer_norm_grad(x, w, mean.double(), rstd, x), TypeError, "mean is")):
        with pytest.raises(error, match=text):
            call()
