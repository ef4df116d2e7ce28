"""Gates of the recurrence that shut: what little is left of a state keeps its bits, on the way there and back."""
import pytest
import torch

from heliox_amd import readout
from readout_util import UNIT

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
F32 = 2.0 ** -24


def near(got, want, dtype, halves, name):
    """Each value to its type's half step and `halves` halves of fp32's, relative to itself."""
    got, want = got.cpu().double(), want.double()
    bound = ((0.0 if dtype is None else UNIT[dtype]) + halves * F32) * want.abs() + 2.0 ** -126
    if dtype is torch.float16:
        bound += 2.0 ** -25
    off = (got - want).abs()
    worst = int((off - bound).argmax())
    assert bool((off <= bound).all()), (name, float(got.flatten()[worst]), float(want.flatten()[worst]))


def resets(batch, time, channels, dtype):
    """States of 1000 that last, but for three steps whose gates shut, from -1 to -25 along the channels."""
    gen = torch.Generator().manual_seed(time)
    gate = 9 + 3 * torch.rand(batch, time, channels, generator=gen)
    at = [time // 4, time // 2, 3 * time // 4]
    gate[:, at] = -1 - 24 * torch.arange(channels) / max(channels - 1, 1) - torch.rand(batch, 3, channels, generator=gen) * 0.5
    state = 1000 * (0.5 + torch.rand(batch, channels, generator=gen))
    last = 0.5 + torch.rand(batch, channels, generator=gen)
    return gate.to(dtype).cuda(), state.cuda(), last.to(dtype).cuda(), at


@pytest.mark.parametrize("batch,time,channels", [(2, 40, 70), (3, 8, 130), (2, 700, 70), (1, 2600, 3), (2, 1100, 9), (170, 90, 33),
                                                 (1, 3000, 129)])
@pytest.mark.parametrize("dtype", TYPES)
def test_what_a_reset_leaves(batch, time, channels, dtype):
    """Without inputs every value is a product.  An open step rounds once; z's own error counts 1e-4 times there.
    A shut step's a takes e^gate (its argument, up to 37, is off by half a step of 32 and by the constant's own error:
    28 halves in all, the instruction's unit 2), 1 + e, its reciprocal (2) and two products: 36.  Runs join in at most 64 products.  dgate is a value of
    the way there times one of the way back, and three more products."""
    gate, state, last, at = resets(batch, time, channels, dtype)
    x, do = torch.zeros_like(gate), torch.zeros_like(gate)
    do[:, -1] = last
    a, z = (1 / (1 + torch.exp(s * gate.cpu().double())) for s in (-1, 1))
    want = a.cumprod(1) * state.cpu().double()[:, None]
    before = torch.cat([state.cpu().double()[:, None], want[:, :-1]], 1)
    back = torch.cat([a[:, 1:].flip(1).cumprod(1).flip(1), torch.ones(batch, 1, channels)], 1) * last.cpu().double()[:, None]
    o, end = readout.gated_recurrence(x, gate, initial_state=state)
    dx, dgate, dinitial = readout.gated_recurrence_grad(x, gate, do, initial_state=state)
    torch.cuda.synchronize()
    halves = time + 3 * 36 + 64
    near(o, want, dtype, halves, "o")
    near(end, want[:, -1], None, halves, "end")
    near(dinitial, a[:, 0] * back[:, 0], None, halves, "dinitial")
    near(dx[:, at], (z * back)[:, at], dtype, halves + 40, "dx")
    near(dgate[:, at], (a * z * back * before)[:, at], dtype, 2 * halves + 40, "dgate")


@pytest.mark.parametrize("channels", [64, 70])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_single_step(channels, dtype):
    gate, state, _, _ = resets(5, 8, channels, dtype)
    gate = gate[:, 4].contiguous()
    want = state.cpu().double() / (1 + torch.exp(-gate.cpu().double()))
    o = readout.gated_recurrence_step(torch.zeros_like(gate), gate, state)
    torch.cuda.synchronize()
    near(o, want, dtype, 40, "o")
    near(state, want, None, 40, "state")


def test_around_where_gates_shut():
    """From -3 to 3: a of e^gate (its argument 3 halves, the constant's error 1, the instruction's unit 2), 1 + e, its
    reciprocal (2) and a product is off by 10 halves of itself; 1 - z, z being at most 0.73 and off by 4 halves,
    by 4 * 0.73 / 0.27 = 11.  One product more."""
    gate = torch.linspace(-3, 3, 100_001)[None].cuda()
    state = torch.full_like(gate, 1000.0)
    want = 1000 / (1 + torch.exp(-gate.cpu().double()))
    o, end = readout.gated_recurrence(torch.zeros_like(gate)[None], gate[None], initial_state=state)
    readout.gated_recurrence_step(torch.zeros_like(gate), gate, state)
    torch.cuda.synchronize()
    for got in (o[0], end, state):
        near(got, want, None, 12, "a step")


@pytest.mark.parametrize("dtype", TYPES)
def test_a_step_is_what_a_run_makes_of_it(dtype):
    """One step and a sequence of one, over all gates: the step's state moves by the same three roundings, the run's value is
    P h + Y, two more.  (Sizes of both terms, which may cancel.)"""
    gate = torch.linspace(-100, 100, 4001)[None, None].to(dtype).cuda()
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(1, 1, 4001, generator=gen).to(dtype).cuda()
    state = (1000 * torch.randn(1, 4001, generator=gen)).cuda()
    a = 1 / (1 + torch.exp(-gate[0].cpu().double()))
    size = a * state.cpu().double().abs() + (1 - a) * x[0].cpu().double().abs()
    _, end = readout.gated_recurrence(x, gate, initial_state=state)
    readout.gated_recurrence_step(x[:, 0], gate[:, 0], state)
    torch.cuda.synchronize()
    assert bool(((state.cpu().double() - end.cpu().double()).abs() <= 8 * F32 * size + 2.0 ** -126).all())


def test_neighbours_do_not_turn_a_bit():
    """A channel's values do not depend on whether gates beside it shut."""
    gen = torch.Generator().manual_seed(1)
    x, gate, do = (torch.randn(2, 300, 64, generator=gen).cuda() for _ in range(3))
    gate += 4.0
    want = *readout.gated_recurrence(x, gate), *readout.gated_recurrence_grad(x, gate, do)[:2]
    gate[:, ::3, 5] = -7.0
    got = *readout.gated_recurrence(x, gate), *readout.gated_recurrence_grad(x, gate, do)[:2]
    keep = torch.arange(64) != 5
    assert all(torch.equal(a[..., keep], b[..., keep]) and not torch.equal(a, b) for a, b in zip(want, got))
