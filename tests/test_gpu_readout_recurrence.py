"""The gated recurrence, its gradient and its single step on the GPU against the recurrence in 64 bits."""
import pytest
import torch

from heliox_amd import HelioxError, readout
from readout_util import UNIT, captured

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
F32 = 2.0 ** -24


def recurrence(x, gate, initial=None, lengths=None, do=None, dend=None):
    """Step by step, float64 on the CPU."""
    x, gate = x.detach().cpu().double(), gate.detach().cpu().double()
    a, z = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(gate))
    batch, steps, c = x.shape
    end = torch.zeros(batch, c, dtype=torch.float64) if initial is None else initial.cpu().double().clone()
    o, dx, dgate = (torch.zeros_like(x) for _ in range(3))
    do = None if do is None else do.cpu()
    back = torch.zeros_like(end) if dend is None else dend.cpu().double().clone()
    lengths = torch.full((batch,), steps) if lengths is None else lengths.cpu().long()
    before = torch.zeros_like(x)
    for t in range(steps):
        live = lengths > t
        before[live, t] = end[live]
        end[live] = a[live, t] * end[live] + z[live, t] * x[live, t]
        o[live, t] = end[live]
    for t in reversed(range(steps if do is not None else 0)):
        live = lengths > t
        l = back[live] + do[live, t].cpu().double()
        dx[live, t] = z[live, t] * l
        dgate[live, t] = a[live, t] * z[live, t] * l * (before[live, t] - x[live, t])
        back[live] = a[live, t] * l
    return o, end, dx, dgate, back


def inputs(seed, batch, time, channels, dtype, memory=1000.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(batch, time, channels, generator=gen)
    keep = torch.log(4.0 * (memory / 4.0) ** (torch.arange(channels) / max(channels - 1, 1)) - 1.0)
    gate = keep + torch.randn(batch, time, channels, generator=gen)
    do = torch.randn(batch, time, channels, generator=gen)
    state, dstate = torch.randn(2, batch, channels, generator=gen).cuda()
    return [t.to(dtype).cuda() for t in (x, gate, do)] + [state, dstate]


def close(got, want, dtype, name):
    """To the type's half step of each value, and fp32's errors, of the tensor's largest values: an
    opening z has at most four roundings and e^gate's error, whose argument of up to 16 carries
    half a step of 32 (32 in all); a state forgets its roundings as it forgets its inputs, one a step against z:
    at most 1 / z of them, that add up like the square root (32 for 1000 steps); runs' products
    and joins add fewer than 64.  dgate takes three such values."""
    got, want = got.cpu().double(), want.double()
    assert got.shape == want.shape and bool(torch.isfinite(got).all())
    if not want.numel():
        return
    unit = 0.0 if dtype is None else UNIT[dtype]
    near = unit * want.abs() + 128 * F32 * (3 if name == "dgate" else 1) * float(want.abs().max())
    if dtype == torch.float16:
        near += 2.0 ** -25
    off = (got - want).abs() - near
    assert bool((off <= 0).all()), (name, float(off.max()))


def check(x, gate, do, state=None, lengths=None, dstate=None):
    want = recurrence(x, gate, state, lengths, do, dstate)
    o, end = readout.gated_recurrence(x, gate, initial_state=state, lengths=lengths)
    dx, dgate, dinitial = readout.gated_recurrence_grad(x, gate, do, initial_state=state, lengths=lengths, dstate=dstate)
    torch.cuda.synchronize()
    assert o.dtype == dx.dtype == dgate.dtype == x.dtype and end.dtype == torch.float32
    assert (dinitial is None) == (state is None)
    for got, exact, name, kind in zip((o, end, dx, dgate, dinitial), want, ("o", "end", "dx", "dgate", "dinitial"),
                                      (x.dtype, None, x.dtype, x.dtype, None)):
        if got is not None:
            close(got, exact, kind, name)
    for i, n in enumerate([] if lengths is None else lengths.tolist()):
        assert all(bool((t[i, n:] == 0).all()) for t in (o, dx, dgate))


@pytest.mark.parametrize("time", [0, 1, 2, 7, 8, 9, 63, 64, 65, 127, 128, 129, 255, 300, 700])
@pytest.mark.parametrize("dtype", TYPES)
def test_lengths_of_time(time, dtype):
    x, gate, do, state, dstate = inputs(time, 2, time, 70, dtype)
    check(x, gate, do, state, None, dstate)


@pytest.mark.parametrize("channels", [1, 2, 3, 4, 5, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 200, 601])
@pytest.mark.parametrize("dtype", TYPES)
def test_channels(channels, dtype):
    x, gate, do, state, dstate = inputs(channels, 3, 90, channels, dtype)
    check(x, gate, do, state, None, dstate)


@pytest.mark.parametrize("batch,time,channels", [(1, 5000, 40), (2, 2500, 130), (130, 150, 3), (40, 140, 513), (2, 9000, 3),
                                                 (170, 2100, 2), (2, 2500, 14), (170, 1050, 9)])
def test_cut_and_whole(batch, time, channels):
    """Few chains, cut into many segments, and enough for a workgroup to walk along each."""
    x, gate, do, state, dstate = inputs(0, batch, time, channels, torch.float32)
    check(x, gate, do, state, None, dstate)


@pytest.mark.parametrize("dtype", TYPES)
def test_without_states(dtype):
    x, gate, do, _, _ = inputs(1, 2, 200, 33, dtype)
    check(x, gate, do)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [5, 150])
def test_ragged(dtype, channels):
    """What lies past a sequence's end is no number, and reaches nothing."""
    x, gate, do, state, dstate = inputs(2, 9, 300, channels, dtype)
    lengths = torch.tensor([300, 0, 1, 7, 8, 64, 65, 128, 299], dtype=torch.int32).cuda()
    for t in (x, gate, do):
        for i, n in enumerate(lengths.tolist()):
            t[i, n:] = float("nan")
    check(x, gate, do, state, lengths, dstate)


def test_views():
    """Inputs side by side in one array, time before batch, rows at odd addresses."""
    gen = torch.Generator().manual_seed(3)
    one = torch.randn(150, 4, 3 * 77 + 1, generator=gen).to(torch.bfloat16).cuda().transpose(0, 1)
    x, gate, do = one[..., 1:78], one[..., 78:155], one[..., 155:]
    check(x, gate, do)
    check(x.transpose(1, 2).contiguous().transpose(1, 2), gate, do)
    check(x[:, ::3], gate[:, ::3], do[:, ::3])
    same = torch.randn(1, 1, 20, generator=gen).cuda().expand(3, 100, 20)
    check(same, same, same)


def test_gates_that_are_shut_or_open():
    """Gates far out and infinite: the state is kept to the bit, or taken from x."""
    x, gate, do, state, dstate = inputs(4, 2, 150, 64, torch.float32)
    gate[:, :, :16] = float("inf")
    gate[:, :, 16:32] = -float("inf")
    gate[:, :, 32:40] = 95.0
    gate[:, :, 40:48] = -95.0
    check(x, gate, do, state, None, dstate)
    o, end = readout.gated_recurrence(x, gate, initial_state=state)
    assert torch.equal(end[:, :16], state[:, :16]) and torch.equal(o[:, :, 16:32], x[:, :, 16:32])


def test_long_memory_of_constant_gates():
    """An error of the opening that is the same at every step would add up: 1 / z is 3000 steps, the
    sequence 20000."""
    x = torch.ones(1, 20000, 4, device="cuda") * torch.tensor([1.0, 0.5, -3.0, 2.0], device="cuda")
    gate = torch.full((1, 20000, 4), 8.0, device="cuda")
    check(x, gate, torch.ones_like(x))


@pytest.mark.parametrize("channels", [6, 130])
def test_what_is_not_finite_reaches_no_earlier_step(channels):
    x, gate, do, state, _ = inputs(5, 1, 400, channels, torch.float32)
    o, _ = readout.gated_recurrence(x, gate, initial_state=state)
    g = readout.gated_recurrence_grad(x, gate, do, initial_state=state)
    x2, do2 = x.clone(), do.clone()
    x2[0, 201, 1], x2[0, 250, 2] = float("nan"), float("inf")
    o2, _ = readout.gated_recurrence(x2, gate, initial_state=state)
    assert torch.equal(o[0, :201], o2[0, :201]) and torch.equal(o[0, :, 3:], o2[0, :, 3:])
    assert bool(o2[0, 201:, 1].isnan().all()) and not bool(torch.isfinite(o2[0, 250:, 2]).any())
    do2[0, 100, 1] = float("nan")
    g2 = readout.gated_recurrence_grad(x, gate, do2, initial_state=state)
    for whole, hit in zip(g[:2], g2[:2]):
        assert torch.equal(whole[0, 101:], hit[0, 101:]) and torch.equal(whole[0, :, 2:], hit[0, :, 2:])
        assert bool(hit[0, :101, 1].isnan().all())


def test_gradients_against_differences():
    """Central differences of the recurrence in 64 bits around the kernel's inputs."""
    x, gate, do, state, dstate = inputs(6, 2, 70, 9, torch.float32, memory=30.0)
    got = readout.gated_recurrence_grad(x, gate, do, initial_state=state, dstate=dstate)

    def loss(x, gate, state):
        o, end = recurrence(x, gate, state)[:2]
        return float((o * do.cpu().double()).sum() + (end * dstate.cpu().double()).sum())

    for which, grad in enumerate(got):
        args = [t.cpu().double() for t in (x, gate, state)]
        way = torch.randn(grad.shape, generator=torch.Generator().manual_seed(9), dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            moved = list(args)
            moved[which] = args[which] + sign * 1e-4 * way
            ends.append(loss(*moved))
        slope = float((grad.cpu().double() * way).sum())
        assert abs((ends[0] - ends[1]) / 2e-4 - slope) <= 1e-5 * float(grad.cpu().double().norm() * way.norm())


@pytest.mark.parametrize("channels", [1, 3, 4, 500, 1024])
@pytest.mark.parametrize("dtype", TYPES)
def test_steps_are_the_whole(channels, dtype):
    """Step by step in shuffled slots gives the whole sequences' outputs and states."""
    x, gate, _, state, _ = inputs(7, 5, 12, channels, dtype)
    o, end = readout.gated_recurrence(x, gate, initial_state=state)
    want = recurrence(x, gate, state)
    slots = torch.tensor([6, 0, 3, 2, 7], dtype=torch.int32).cuda()
    pool = torch.full((9, channels), 5.0, device="cuda")
    pool[slots.long()] = state
    for t in range(12):
        got = readout.gated_recurrence_step(x[:, t], gate[:, t], pool, slots=slots)
        close(got, want[0][:, t], dtype, "o")
    close(pool[slots.long()], want[1], None, "end")
    rest = torch.ones(9, dtype=torch.bool)
    rest[slots.cpu().long()] = False
    assert bool((pool[rest] == 5.0).all())


def test_rows_without_a_slot():
    x, gate, _, state, _ = inputs(8, 4, 1, 12, torch.float16)
    x[1] = float("nan")
    pool = state.clone()
    slots = torch.tensor([2, -1, 4, 0], dtype=torch.int32).cuda()
    o = readout.gated_recurrence_step(x[:, 0], gate[:, 0], pool, slots=slots)
    assert bool((o[1:3] == 0).all()) and bool((o[0] != 0).any()) and bool((o[3] != 0).any())
    assert torch.equal(pool[[1, 3]], state[[1, 3]]) and not torch.equal(pool[[0, 2]], state[[0, 2]])
    again = state.clone()
    readout.gated_recurrence_step(x[:, 0], gate[:, 0], again)           # row i, slot i
    assert bool(again[1].isnan().all()) and bool(torch.isfinite(again[[0, 2, 3]]).all())


@pytest.mark.parametrize("batch,time,channels", [(2, 900, 40), (3, 20, 40)])
def test_captured(batch, time, channels):
    x, gate, do, state, dstate = inputs(9, batch, time, channels, torch.float32)
    lengths = torch.tensor([time, time // 2, 1][:batch], dtype=torch.int32).cuda()

    def call():
        how = dict(initial_state=state, lengths=lengths)
        return [*readout.gated_recurrence(x, gate, **how), *readout.gated_recurrence_grad(x, gate, do, dstate=dstate, **how)]

    def change(gen):
        for t in (x, gate, do, state):
            t.copy_(torch.randn(t.shape, generator=gen))
        lengths.copy_(torch.randint(0, time + 1, (batch,), generator=gen))

    captured(call, change)


def test_streams_of_their_own():
    x, gate, do, state, _ = inputs(10, 1, 3000, 100, torch.float32)
    want = readout.gated_recurrence(x, gate, initial_state=state)[0]
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            got.append(readout.gated_recurrence(x, gate, initial_state=state)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(want, g) for g in got)


def test_offsets_past_32_bits():
    """The last sequences of 2^32 elements and more."""
    batch, time, channels = 3, 2, 1 << 30
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GiB of device memory")
    x = torch.zeros(batch, time, 1, dtype=torch.float16, device="cuda").expand(batch, time, 8).contiguous()
    wide = torch.empty(batch, time * channels, dtype=torch.float16, device="cuda")
    far = wide.view(batch, time, channels)[..., -8:]
    far.copy_(torch.randn(batch, time, 8, generator=torch.Generator().manual_seed(0)))
    check(far, far, far)


def test_refusals():
    x, gate, do, state, _ = inputs(11, 2, 5, 6, torch.float32)
    step = readout.gated_recurrence_step
    for call, error, text in (
            (lambda: readout.gated_recurrence(x, gate[:, :4]), ValueError, "gate has shape"),
            (lambda: readout.gated_recurrence(x, gate.half()), TypeError, "gate is"),
            (lambda: readout.gated_recurrence(x.double(), gate.double()), TypeError, "not float32"),
            (lambda: readout.gated_recurrence(x[0], gate[0]), ValueError, "batch, time, channels"),
            (lambda: readout.gated_recurrence(x[..., :0], gate[..., :0]), ValueError, "channel"),
            (lambda: readout.gated_recurrence(x, gate.cpu()), ValueError, "GPU"),
            (lambda: readout.gated_recurrence(x, gate, initial_state=state[:1]), ValueError, "initial_state has shape"),
            (lambda: readout.gated_recurrence(x, gate, initial_state=state.half()), TypeError, "initial_state is"),
            (lambda: readout.gated_recurrence(x, gate, lengths=torch.ones(2).cuda()), TypeError, "lengths is"),
            (lambda: readout.gated_recurrence(x.clone().requires_grad_(), gate), ValueError, "records no graph"),
            (lambda: readout.gated_recurrence_grad(x, gate, do[:1]), ValueError, "do has shape"),
            (lambda: readout.gated_recurrence_grad(x, gate, do.half()), TypeError, "do is"),
            (lambda: readout.gated_recurrence_grad(x, gate, do, dstate=state[0]), ValueError, "dstate has shape"),
            (lambda: step(x, gate, state), ValueError, "batch, channels"),
            (lambda: step(x[:, 0], gate[:, 0], state.half()), TypeError, "state has to be"),
            (lambda: step(x[:, 0], gate[:, 0], state.t().contiguous().t()), TypeError, "contiguous"),
            (lambda: step(x[:, 0], gate[:, 0], state[:, :5].contiguous()), ValueError, "state has shape"),
            (lambda: step(x[:, 0], gate[:, 0], state[:1]), HelioxError, "only 1 states")):
        with pytest.raises(error, match=text):
            call()
