"""The loss against a teacher's top logits and the drawing of answers on the GPU, against
64-bit results row by row."""
import math

import pytest
import torch

import readout_util as ref
from heliox_amd import readout

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
F32 = ref.UNIT[torch.float32]


# ------------------------------------------------------------------------- distillation
def problem(seed, dtype, rows, vocab, top, tau, index_type=torch.int32, scale=3.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=gen) * scale
    full = 0.6 * x + torch.randn(rows, vocab, generator=gen)
    t, index = torch.topk(full, top, dim=1)
    lse = torch.logsumexp(full / tau, 1)
    weight = torch.rand(rows, generator=gen) + 0.5
    return x.to(dtype).cuda(), index.to(index_type).cuda(), t.to(dtype).cuda(), lse.cuda(), weight.cuda()


# Losses are fp32: each of the terms p (log p - log q) is off by a few units times the largest
# logarithm (under 2^6), and they are as large as the loss together; gradients are rounded once
# to their type, before it good to 2^6 fp32 units of the probabilities that they are made of.
def loss_bound(want):
    return 2 ** 8 * F32 * want.abs().clamp(min=1.0)


def grad_bound(dtype):
    return 2 ** 8 * F32 + (ref.UNIT[dtype] if dtype != torch.float32 else 0.0)


def check(x, index, t, tau, lse, weight, dtype):
    print(f"case distill {dtype} {tuple(x.shape)} top={index.shape[1]} tau={tau} rest={lse is not None}", flush=True)
    want, dwant = ref.distill(x, index, t, tau, lse, weight)
    loss = readout.distill_loss(x, index, t, temperature=tau, teacher_lse=lse)
    both, grad = readout.distill_loss_grad(x, index, t, temperature=tau, teacher_lse=lse, weight=weight)
    torch.cuda.synchronize()
    assert torch.equal(loss, both) and loss.dtype == torch.float32 and grad.dtype == dtype
    assert bool(((loss.cpu().double() - want).abs() <= tau * tau * loss_bound(want / (tau * tau))).all())
    assert ref.rel(grad, dwant) <= grad_bound(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("rows,vocab,top,tau", [
    (1, 1, 1, 1.0), (3, 2, 1, 1.0), (5, 17, 5, 2.0), (4, 255, 255, 1.0), (9, 1000, 5, 2.0), (2, 1023, 64, 0.5),
    (3, 4097, 33, 3.0), (2, 50021, 100, 1.0), (2, 131072, 64, 1.0), (1, 300001, 7, 1.0)])
def test_distill(dtype, rest, rows, vocab, top, tau):
    x, index, t, lse, weight = problem(rows + vocab, dtype, rows, vocab, top, tau)
    if top == vocab:
        rest = False            # nothing beside the entries
    check(x, index, t, tau, lse if rest else None, weight, dtype)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("index_type", [torch.int32, torch.int64])
def test_distill_absent_and_double_entries(rest, index_type):
    x, index, t, lse, weight = problem(3, torch.float32, 6, 500, 12, 1.0, index_type)
    lse = lse + 0.5             # room for the entries that come twice
    index[0, 3:] = -1
    index[1, :] = -1            # a row without a teacher
    index[2, 5] = 500           # not a place
    index[3, 7] = index[3, 2]
    index[3, 9] = index[3, 2]
    t[4, 1] = -math.inf
    check(x, index, t, 1.0, lse if rest else None, weight, torch.float32)
    loss, grad = readout.distill_loss_grad(x, index, t, teacher_lse=lse if rest else None)
    assert float(loss[1]) == 0 and not grad[1].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("low", ["inf", "lowest"])
def test_distill_masked_student(dtype, low):
    """Places that the student's mask rules out, with infinity or with the type's lowest value."""
    x, index, t, lse, weight = problem(4, dtype, 4, 700, 9, 1.0)
    ruled = torch.zeros(700, dtype=torch.bool, device="cuda")
    ruled[::3] = True
    ruled[index.long().unique()] = False
    x[:, ruled] = -math.inf if low == "inf" else torch.finfo(dtype).min
    check(x, index, t, 1.0, lse, weight, dtype)
    _, grad = readout.distill_loss_grad(x, index, t, teacher_lse=lse)
    assert not grad[:, ruled].any()
    # an entry that the mask rules out: an infinite loss, a finite gradient
    x[0, int(index[0, 0])] = -math.inf
    loss, grad = readout.distill_loss_grad(x, index, t)
    assert math.isinf(float(loss[0])) and bool(torch.isfinite(grad).all())


def test_distill_teacher_of_nothing_but_minus_infinity():
    x, index, t, lse, _ = problem(5, torch.float32, 2, 64, 4, 1.0)
    t[0] = -math.inf
    loss, grad = readout.distill_loss_grad(x, index, t)
    assert float(loss[0]) == 0 and not grad[0].any() and float(loss[1]) > 0


@pytest.mark.parametrize("dtype", TYPES)
def test_distill_strides_and_in_place(dtype):
    gen = torch.Generator().manual_seed(6)
    wide = (torch.randn(7, 1205, generator=gen) * 2).to(dtype).cuda()
    x = wide[:, 3:1204]         # rows at odd addresses
    index = torch.randint(0, 1201, (7, 20), generator=gen).cuda()[:, ::2]
    t = torch.randn(10, 7, generator=gen).to(torch.float32).cuda().t()
    want, dwant = ref.distill(x, index, t, 1.0)
    kept = wide.clone()
    loss, grad = readout.distill_loss_grad(x, index, t, out=x)
    assert grad.data_ptr() == x.data_ptr()
    assert torch.equal(wide[:, :3], kept[:, :3]) and torch.equal(wide[:, 1204:], kept[:, 1204:])
    assert bool(((loss.cpu().double() - want).abs() <= loss_bound(want)).all())
    assert ref.rel(grad, dwant) <= grad_bound(dtype)


def test_distill_no_entries_or_rows():
    x = torch.randn(3, 50, device="cuda")
    loss, grad = readout.distill_loss_grad(x, torch.zeros(3, 0, dtype=torch.int32, device="cuda"),
                                           torch.zeros(3, 0, device="cuda"))
    assert not loss.any() and not grad.any()
    loss, grad = readout.distill_loss_grad(x[:0], torch.zeros(0, 4, dtype=torch.int32, device="cuda"),
                                           torch.zeros(0, 4, device="cuda"))
    assert loss.shape == (0,) and grad.shape == (0, 50)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("tau", [1.0, 2.5])
def test_distill_gradient_against_differences(rest, tau):
    """Central differences along a random way: their own error is step^2 / 6 times a third
    derivative that is under 1 for |way| 1; the losses' rounding is divided by the step."""
    x, index, t, lse, _ = problem(7, torch.float32, 5, 300, 11, tau)
    lse = lse if rest else None
    _, grad = readout.distill_loss_grad(x, index, t, temperature=tau, teacher_lse=lse)
    way = torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).cuda()
    way = way / way.norm(dim=1, keepdim=True)
    step = 0.05
    up, down = (readout.distill_loss(x + s * way, index, t, temperature=tau, teacher_lse=lse) for s in (step, -step))
    diff = (up.double() - down.double()) / (2 * step)
    exact = (grad.double() * way.double()).sum(1)
    noise = tau * tau * loss_bound(up.double() / (tau * tau)) / step
    assert bool(((diff - exact).abs() <= noise + step * step / 6).all())


def test_distill_same_bits():
    x, index, t, lse, weight = problem(8, torch.bfloat16, 40, 20001, 30, 1.0)
    one = readout.distill_loss_grad(x, index, t, teacher_lse=lse, weight=weight)
    two = readout.distill_loss_grad(x, index, t, teacher_lse=lse, weight=weight)
    assert all(torch.equal(a, b) for a, b in zip(one, two))


# ----------------------------------------------------------------------------- sampling
def check_draws(x, u, temperature, top_k, top_p, min_p):
    """Every token stays and lies where u of the kept mass falls, but for the share by which the
    library's fp32 weights can shift a sum (2^4 units: the weights' own rounding)."""
    rows = x.shape[0]
    token, logprob = readout.sample(x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    torch.cuda.synchronize()
    at = lambda s, i: float(s[i]) if isinstance(s, torch.Tensor) else s  # noqa: E731
    for i in range(rows):
        p, floor = at(top_p, i), at(min_p, i)
        slack = 2 ** 4 * F32
        j = int(token[i])
        m, stays = ref.masses(x[i], at(temperature, i), int(at(top_k, i)), p, floor)
        if not stays[j]:        # a place at the edge of top_p or min_p, moved by a rounding
            m, stays = ref.masses(x[i], at(temperature, i), int(at(top_k, i)), min(1.0, p * (1 + slack)) if p < 1 else p,
                                  floor * (1 - slack))
        assert stays[j], (i, j)
        kept = torch.where(stays, m, 0.0)
        total = float(kept.sum())
        before = float(kept[:j].sum())
        aim = float(u[i]) * total
        edge = slack * total + 1.0 + (float(kept[stays].min()) if p < 1 or floor > 0 else 0.0)
        assert before - edge <= aim <= before + float(kept[j]) + edge, (i, j, before, aim)
        want = math.log(float(kept[j]) / total)
        assert abs(float(logprob[i]) - want) <= 2 ** 5 * F32 * max(1.0, abs(want)) + edge / total


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 257, 1000, 1025, 5003, 32000, 131072, 200003])
def test_sample(dtype, vocab):
    print(f"case sample {dtype} vocab={vocab}", flush=True)
    gen = torch.Generator().manual_seed(vocab)
    rows = 12
    x = (torch.randn(rows, vocab, generator=gen) * 3).to(dtype).cuda()
    u = torch.rand(rows, generator=gen).cuda()
    pick = lambda *v: torch.tensor(v)[torch.randint(len(v), (rows,), generator=gen)].cuda()  # noqa: E731
    check_draws(x, u, 1.0, 0, 1.0, 0.0)
    check_draws(x, u, 0.8, 40, 0.9, 0.02)
    check_draws(x, u, pick(0.0, 0.5, 1.0, 2.0), pick(0, 1, 7, 100, vocab + 5).to(torch.int32), pick(0.0, 0.3, 0.9, 1.0),
                pick(0.0, 0.05, 1.0))


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_ties_go_to_the_lowest_index(dtype):
    x = torch.zeros(6, 1000, dtype=dtype, device="cuda")
    u = torch.tensor([0.0, 0.25, 0.5, 0.999, 0.1, 0.99], device="cuda")
    token, logprob = readout.sample(x, u)
    assert token.tolist() == [0, 250, 500, 999, 100, 990]
    token, logprob = readout.sample(x, u, top_k=10)
    assert token.tolist() == [0, 2, 5, 9, 1, 9]
    assert torch.allclose(logprob, torch.full_like(logprob, -math.log(10)), atol=1e-6)
    # 0.0125 of 1000 equal places: 13 of them are the fewest that hold as much
    token, logprob = readout.sample(x, u, top_p=0.0125)
    assert token.tolist() == [0, 3, 6, 12, 1, 12]
    # the fp32 number nearest to 0.1 is over a tenth of the 20 that top_k leaves: three places hold as much
    token, _ = readout.sample(x, u, top_k=20, top_p=0.1)
    assert token.tolist() == [0, 0, 1, 2, 0, 2]
    assert readout.sample(x, u, temperature=0.0)[0].tolist() == [0] * 6
    x[:, 700] = 1
    x[:, 800] = 1
    token, logprob = readout.sample(x, u, temperature=0.0)
    assert token.tolist() == [700] * 6 and not logprob.any()
    token, _ = readout.sample(x, u, top_k=2)
    assert token.tolist() == [700, 700, 800, 800, 700, 800]
    token, _ = readout.sample(x, u, min_p=1.0)
    assert token.tolist() == [700, 700, 800, 800, 700, 800]
    token, _ = readout.sample(x, u, top_k=4)
    assert set(token.tolist()) <= {0, 1, 700, 800}


def test_sample_signed_zeros_tie():
    x = torch.zeros(1, 100, device="cuda")
    x[0, ::2] = -0.0
    u = torch.tensor([0.9], device="cuda")
    assert readout.sample(x, u, top_k=5)[0].tolist() == [4]


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_masks_infinities_and_nan(dtype):
    x = torch.randn(7, 300, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    u = torch.linspace(0, 0.99, 7).cuda()
    x[0] = -math.inf                            # nothing left
    x[1] = -math.inf
    x[1, 123] = -5                              # one place left
    x[2] = torch.finfo(dtype).min
    x[2, 7] = 1
    x[3, ::2] = math.nan
    x[4] = math.nan
    x[5, 50], x[5, 60] = math.inf, math.inf
    x[6] = torch.finfo(dtype).min               # all ruled out alike: all alike
    for how in ({}, {"top_k": 5}, {"top_p": 0.7}, {"min_p": 0.1}, {"temperature": 0.0},
                {"top_k": 50, "top_p": 0.9, "min_p": 0.01, "temperature": 0.7}):
        token, logprob = readout.sample(x, u, **how)
        token = token.tolist()
        assert token[0] == -1 and token[4] == -1 and float(logprob[0]) == -math.inf
        assert token[1] == 123 and float(logprob[1]) == 0
        assert token[2] == 7
        assert token[3] % 2 == 1
        assert token[5] in (50, 60)
        assert 0 <= token[6] < 300


def test_sample_small_temperatures_and_edges_of_u():
    x = torch.randn(4, 500, generator=torch.Generator().manual_seed(2)).cuda()
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 0.5], device="cuda")
    token, _ = readout.sample(x, u, temperature=1e-40)
    assert token.tolist() == x.argmax(1).tolist()
    token, logprob = readout.sample(x, u)
    assert int(token[0]) == 0 and int(token[1]) == 499 and int(token[2]) == 499
    assert bool((logprob < 0).all())


def test_sample_frequencies():
    """100,000 draws of one row: counts within five standard deviations of the probabilities."""
    n, p = 100_000, torch.tensor([0.5, 0.25, 0.125, 0.0625, 0.0625])
    x = p.log().expand(n, 5).cuda()
    u = torch.rand(n, generator=torch.Generator().manual_seed(3)).cuda()
    token, _ = readout.sample(x, u)
    count = torch.bincount(token, minlength=5).cpu().double()
    assert bool(((count - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all())
    kept = p[:3] / p[:3].sum()
    token, _ = readout.sample(x, u, top_p=0.8)
    count = torch.bincount(token, minlength=5).cpu().double()
    assert bool(((count[:3] - n * kept).abs() <= 5 * (n * kept * (1 - kept)).sqrt()).all()) and not count[3:].any()


def test_sample_strides():
    wide = torch.randn(9, 1301, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    u = torch.rand(9, generator=torch.Generator().manual_seed(5)).cuda()
    x = wide[:, 1:1300]
    a, b = readout.sample(x, u, top_k=30, top_p=0.8), readout.sample(x.contiguous(), u, top_k=30, top_p=0.8)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    check_draws(x, u, 1.0, 30, 0.8, 0.0)
    flipped = x.t().contiguous().t()            # last dimension not contiguous
    assert all(torch.equal(p, q) for p, q in zip(readout.sample(flipped, u, top_k=30, top_p=0.8), a))


def test_rows_more_than_32_bits_apart():
    far = 2 ** 31 + 24
    space = torch.empty(far + 5000, dtype=torch.bfloat16, device="cuda")
    x, index, t, lse, weight = problem(9, torch.bfloat16, 2, 5000, 12, 1.0)
    apart = space.as_strided(x.shape, (far, 1))
    apart.copy_(x)
    near = readout.distill_loss_grad(x, index, t, teacher_lse=lse, weight=weight)
    u = torch.tensor([0.3, 0.8], device="cuda")
    drawn = readout.sample(x, u, top_p=0.9)
    assert all(torch.equal(a, b) for a, b in zip(readout.sample(apart, u, top_p=0.9), drawn))
    loss, grad = readout.distill_loss_grad(apart, index, t, teacher_lse=lse, weight=weight, out=apart)
    assert torch.equal(loss, near[0]) and torch.equal(grad, near[1])


# ---------------------------------------------------------- distillation, students far from the teacher
def sure(seed, dtype, gap, tau, rows=3, vocab=203, top=5, masked=None, below=True):
    """Students whose other places lie `gap` temperatures under their entries (below) or over them;
    the teacher has a tenth of its mass beside the entries."""
    gen = torch.Generator().manual_seed(seed)
    index = torch.stack([torch.randperm(vocab, generator=gen)[:top] for _ in range(rows)])
    x = torch.randn(rows, vocab, generator=gen) * tau - (gap * tau if below else 0.0)
    x.scatter_(1, index, torch.randn(rows, top, generator=gen) * tau - (0.0 if below else gap * tau))
    if masked is not None:
        ruled = torch.arange(vocab) % 3 == 0
        ruled[index.unique()] = False
        x[:, ruled] = -math.inf if masked == "inf" else torch.finfo(dtype).min
    t = torch.randn(rows, top, generator=gen).to(dtype)
    lse = torch.logsumexp(t.double() / tau, 1) - math.log(0.9)
    return x.to(dtype).cuda(), index.to(torch.int32).cuda(), t.cuda(), lse.float().cuda()


def check_sure(x, index, t, tau, lse, weight, dtype):
    """Losses as everywhere; gradients row by row, the entries and the others each by themselves."""
    want, dwant = ref.distill(x, index, t, tau, lse, weight)
    loss, grad = readout.distill_loss_grad(x, index, t, temperature=tau, teacher_lse=lse, weight=weight)
    assert bool(torch.isfinite(dwant).all()) and bool(torch.isfinite(grad).all())
    assert torch.equal(loss, readout.distill_loss(x, index, t, temperature=tau, teacher_lse=lse))
    assert bool(((loss.cpu().double() - want).abs() <= tau * tau * loss_bound(want / (tau * tau))).all()), (loss, want)
    entries = torch.zeros(x.shape, dtype=torch.bool).scatter_(1, index.cpu().long(), True)
    for part in (entries, ~entries):
        got, exact = (torch.where(part, g.cpu().double(), 0.0) for g in (grad, dwant))
        assert bool(((got - exact).norm(dim=1) <= grad_bound(dtype) * exact.norm(dim=1)).all()), (got - exact).norm(dim=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tau", [0.25, 0.5, 1.0, 2.0, 4.0])
@pytest.mark.parametrize("gap", [20, 46, 60, 87, 90, 95, 100, 104, 200, 400, 700])
def test_distill_the_rest_of_a_sure_student(dtype, tau, gap):
    print(f"case sure student {dtype} gap={gap} tau={tau}", flush=True)
    weight = torch.tensor([16.0, 256.0, 1000.0], device="cuda")
    for masked in (None, "inf", "lowest"):
        x, index, t, lse = sure(gap, dtype, gap, tau, masked=masked)
        check_sure(x, index, t, tau, lse, weight, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gap", [30, 100, 400])
def test_distill_a_student_sure_of_other_places(dtype, gap):
    x, index, t, lse = sure(gap, dtype, gap, 1.0, below=False)
    check_sure(x, index, t, 1.0, lse, torch.tensor([16.0, 256.0, 1000.0], device="cuda"), dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_distill_entries_twice_and_absent_beside_a_far_rest(dtype):
    x, index, t, lse = sure(5, dtype, 100, 1.0, rows=4)
    lse = lse + 1.0                   # room for an entry that comes twice
    index[0, 3] = index[0, 1]
    index[1, 2] = -1
    index[2, 4] = index[2, 0]
    index[2, 1] = 203
    want, dwant = ref.distill(x, index, t, 1.0, lse)
    loss, grad = readout.distill_loss_grad(x, index, t, teacher_lse=lse)
    assert bool(((loss.cpu().double() - want).abs() <= loss_bound(want)).all())
    assert bool(((grad.cpu().double() - dwant).norm(dim=1) <= grad_bound(dtype) * dwant.norm(dim=1)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("low", ["inf", "lowest"])
def test_distill_nothing_left_beside_the_entries(dtype, low):
    """Every other place is masked: their class is not there, and they have no gradient."""
    x, index, t, lse = sure(6, dtype, 0, 1.0)
    others = torch.ones_like(x, dtype=torch.bool).scatter_(1, index.long(), False)
    x[others] = -math.inf if low == "inf" else torch.finfo(dtype).min
    want, dwant = ref.distill(x, index, t, 1.0, lse)
    loss, grad = readout.distill_loss_grad(x, index, t, teacher_lse=lse)
    assert bool(((loss.cpu().double() - want).abs() <= loss_bound(want)).all())
    assert not grad[others].any() and ref.rel(grad, dwant) <= grad_bound(dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_distill_temperatures_at_the_ends(dtype):
    """The coldest student is its largest logit, the hottest knows nothing: finite either way."""
    x, index, t, lse, weight = problem(12, dtype, 3, 300, 5, 1.0)
    x = x.float().cummax(1).values + 0.125 * torch.arange(300, device="cuda")     # one largest, the last
    x = x.to(dtype)
    index[:, 0] = 299
    loss, grad = readout.distill_loss_grad(x, index, t, temperature=2.0 ** -126)
    assert bool(torch.isfinite(loss).all()) and bool(torch.isfinite(grad).all())
    _, grad = readout.distill_loss_grad(x, index, t, temperature=2.0 ** 126, weight=torch.full_like(weight, 2.0 ** -126))
    assert bool(torch.isfinite(grad).all())
    outside = torch.ones(300, dtype=torch.bool, device="cuda")
    outside[index.long().unique()] = False
    assert torch.allclose(grad.float()[:, outside], torch.full_like(grad.float()[:, outside], 1 / 300), rtol=2 ** -7)


def test_distill_gradients_beside_the_logits():
    """Halves of one array, and an array of its own with rows further apart, are taken; parts are refused."""
    x, index, t, lse, weight = problem(13, torch.float32, 6, 500, 9, 1.0)
    want = readout.distill_loss_grad(x, index, t, teacher_lse=lse, weight=weight)[1]
    both = torch.cat([x, torch.zeros_like(x)], dim=1)
    for out in (both[:, 500:], torch.zeros(6, 777, device="cuda")[:, 5:505]):
        readout.distill_loss_grad(both[:, :500], index, t, teacher_lse=lse, weight=weight, out=out)
        assert torch.equal(out, want) and torch.equal(both[:, :500], x)
    one = x[:1].expand(6, -1)
    for logits, out in ((x, torch.zeros(1, 500, device="cuda").expand(6, -1)), (both[:, :500], both[:, 1:501]), (one, one)):
        with pytest.raises(RuntimeError, match="overlap"):
            readout.distill_loss_grad(logits, index, t, teacher_lse=lse, out=out)
    assert torch.equal(readout.distill_loss_grad(one, index, t)[1], readout.distill_loss_grad(one.contiguous(), index, t)[1])


def test_settings_that_are_no_numbers_are_refused():
    x, index, t, *_ = problem(14, torch.float32, 2, 50, 3, 1.0)
    u = torch.rand(2, device="cuda")
    q = torch.randn(1, 3, 2, 8, device="cuda")
    g = torch.zeros(2, device="cuda")
    bad = [
        (TypeError, lambda: readout.sample(x, u, top_k=50.0)),
        (TypeError, lambda: readout.sample(x, u, top_k="5")),
        (TypeError, lambda: readout.sample(x, u, top_k=None)),
        (ValueError, lambda: readout.sample(x, u, top_k=2 ** 63)),
        (TypeError, lambda: readout.sample(x, u, temperature="1.0")),
        (TypeError, lambda: readout.sample(x, u, top_p=None)),
        (TypeError, lambda: readout.sample(x, u, min_p=[0.1])),
        (ValueError, lambda: readout.sample(x, u, temperature=10 ** 400)),
        (TypeError, lambda: readout.distill_loss(x, index, t, temperature="warm")),
        (ValueError, lambda: readout.distill_loss_grad(x, index, t, temperature=10 ** 400)),
        (TypeError, lambda: readout.linear_attention(q, q, q, g, scale="1")),
        (TypeError, lambda: readout.linear_attention_grad(q, q, q, g, q, scale=[1.0])),
        (ValueError, lambda: readout.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], g, q.new_zeros(1, 2, 8, 8), scale=10 ** 400)),
    ]
    for error, call in bad:
        with pytest.raises(error):
            call()
    import numpy as np
    same = readout.sample(x, u, temperature=0.5, top_k=5, top_p=0.75, min_p=0.25)
    other = readout.sample(x, u, temperature=np.float32(0.5), top_k=np.int64(5), top_p=np.float64(0.75), min_p=np.float32(0.25))
    assert all(torch.equal(a, b) for a, b in zip(same, other))
    assert all(torch.equal(a, b) for a, b in zip(readout.sample(x, u, temperature=1, top_p=1, min_p=0), readout.sample(x, u)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rest", [False, True])
def test_distill_rows_of_half_a_chip(dtype, rest):
    """600 rows take 512 threads each."""
    x, index, t, lse, weight = problem(15, dtype, 600, 5003, 12, 1.0)
    check(x, index, t, 1.0, lse if rest else None, weight, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_many_rows_of_several_turns(dtype):
    """1100 rows take 256 threads each, and a row of 5003 places several turns of them."""
    gen = torch.Generator().manual_seed(16)
    x = (torch.randn(1100, 5003, generator=gen) * 3).to(dtype).cuda()
    u = torch.rand(1100, generator=gen).cuda()
    pick = lambda *v: torch.tensor(v)[torch.randint(len(v), (1100,), generator=gen)].cuda()  # noqa: E731
    check_draws(x, u, pick(0.0, 0.5, 1.0, 2.0), pick(0, 1, 7, 100, 900).to(torch.int32), pick(0.3, 0.9, 1.0), pick(0.0, 0.05))


@pytest.mark.parametrize("vocab", [1000, 600_001])     # the bit map of the latter: over 64 KB of LDS
@pytest.mark.parametrize("rest", [False, True])
def test_distill_captured_into_a_graph(rest, vocab):
    x, index, t, lse, weight = problem(17, torch.bfloat16, 3, vocab, 20, 1.0)
    lse = lse if rest else None
    ref.captured(lambda: (readout.distill_loss(x, index, t, teacher_lse=lse),
                          *readout.distill_loss_grad(x, index, t, teacher_lse=lse, weight=weight)),
                 lambda gen: x.copy_((torch.randn(x.shape, generator=gen) * 3).to(x.dtype)))


@pytest.mark.parametrize("vocab", [1000, 3_000_000])   # the sums by turn of the latter: over 32 KB of LDS
def test_sample_captured_into_a_graph(vocab):
    x = torch.zeros(3, vocab, dtype=torch.bfloat16, device="cuda")
    u = torch.zeros(3, device="cuda")

    def change(gen):
        x.copy_((torch.randn(x.shape, generator=gen) * 3).to(x.dtype))
        u.copy_(torch.rand(3, generator=gen))

    change(torch.Generator().manual_seed(9))
    ref.captured(lambda: (*readout.sample(x, u), *readout.sample(x, u, top_k=30, top_p=0.9), *readout.sample(x, u, top_p=0.8)),
                 change)
