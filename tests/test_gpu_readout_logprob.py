"""Log probabilities of given tokens, entropies, top alternatives and their gradient on the GPU
against the definitions in 64 bits."""
import pytest
import torch

from heliox_amd import HelioxError, readout
from readout_util import UNIT, captured

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
F32 = 2.0 ** -24
INF = float("inf")


def definition(logits, tokens, tau, top):
    x = logits.detach().cpu().double()
    rows, vocab = x.shape
    most = torch.where(x.isnan(), -INF, x).amax(1, keepdim=True)
    z = (x - torch.where(most == -INF, 0.0, most)) / tau      # first: rows of a type's lowest value keep log of their count
    logq = torch.where(most == -INF, -INF, z - torch.logsumexp(z, 1, keepdim=True))
    q = logq.exp()
    entropy = -torch.where(q > 0, q * logq, 0.0).sum(1)
    tokens = tokens.cpu().long()
    there = (tokens >= 0) & (tokens < vocab)
    at = torch.where(there, tokens, 0)
    logprob = torch.where(there, logq[torch.arange(rows), at], 0.0)
    index = torch.sort(torch.where(x.isnan(), -INF, x), dim=1, descending=True, stable=True).indices[:, :top]
    return logq, logprob, entropy, logq.gather(1, index), index


# A thread adds at most 160 weights one after another, whose own errors are below 32 halves of a step
# where they count (e^-20 and smaller ones do not).
SUM = 192 * F32


def same(got, want, size=0.0):
    """Equal, or apart by no more than fp32 sums may be; infinities and NaN where they belong (a logarithm
    of -3.4e38 / 0.3 is an infinity in fp32)."""
    got, want = got.cpu().double(), want.double()
    want = torch.where(torch.isfinite(want.float()), want, want.float().double())
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan())
    plain = torch.isfinite(want)
    assert torch.equal(got[~plain & ~want.isnan()], want[~plain & ~want.isnan()])
    off = (got - want).abs()[plain] - (SUM * (1 + size) + 2 * F32 * want.abs()[plain])
    assert not off.numel() or float(off.max()) <= 0, float(off.max())


def check(logits, tokens, tau=1.0, top=0, finite=True):
    logq, logprob, entropy, top_logprob, index = definition(logits, tokens, tau, top)
    got = readout.token_logprobs(logits, tokens, temperature=tau, top=top)
    torch.cuda.synchronize()
    assert torch.equal(got.top_index.cpu(), index)
    same(got.logprob, logprob)
    # both of its terms are at most log(vocab) and the spread of what counts
    same(got.entropy, entropy, size=2 * float(torch.log(torch.tensor(float(logits.shape[1])))) + 1)
    same(got.top_logprob, top_logprob)
    if finite:
        m = logits.cpu().double().amax(1)
        assert torch.equal(got.stats[:, 0].cpu().double(), m)
        same(got.stats[:, 1], torch.logsumexp((logits.cpu().double() - torch.where(m == -INF, 0.0, m)[:, None]) / tau, 1))
    return got


def check_grad(logits, tokens, tau, dlogprob, dentropy, out=None):
    logq, _, entropy, _, _ = definition(logits, tokens, tau, 0)
    rows, vocab = logits.shape
    got = readout.token_logprobs(logits, tokens, temperature=tau)
    grad = readout.token_logprobs_grad(logits, tokens, got, dlogprob, dentropy, temperature=tau, out=out)
    tokens = tokens.cpu().long()
    there = (tokens >= 0) & (tokens < vocab)
    pull = torch.zeros(rows, dtype=torch.float64) if dlogprob is None else torch.where(there, dlogprob.cpu().double(), 0.0)
    turn = torch.zeros(rows, dtype=torch.float64) if dentropy is None else dentropy.cpu().double()
    q, gain = logq.exp(), torch.where(logq > -INF, logq, 0.0)
    want = -q * (pull[:, None] + turn[:, None] * (gain + entropy[:, None]))
    hit = torch.zeros_like(q)
    hit[torch.arange(rows), torch.where(there, tokens, 0)] = 1.0
    want = (want + hit * pull[:, None]) / tau
    # q is off by what log z and the logarithms are, both terms by as much of themselves; at the token
    # 1 - q is off by q's error
    spread = 2 * SUM * (1 + gain.abs().clamp(max=200.0) / 32)
    size = 2 * float(torch.log(torch.tensor(float(vocab)))) + 2
    near = q * (pull.abs()[:, None] * (1 + hit) + turn.abs()[:, None] * (gain.abs() + entropy[:, None] + size)) * spread / tau
    near += UNIT[logits.dtype] * want.abs() + F32 * pull.abs()[:, None] * hit * 4 / tau
    if logits.dtype == torch.float16:
        near += 2.0 ** -25
    near += 2.0 ** -126                    # weights of the exponential's instruction end there
    off = (grad.cpu().double() - want).abs() - near
    assert grad.dtype == logits.dtype and float(off.max()) <= 0, float(off.max())
    return grad


def normal(seed, *shape, dtype=torch.float32, scale=3.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def some(seed, rows, vocab, dtype=torch.int64):
    return torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("vocab", [1, 2, 3, 4, 5, 7, 8, 9, 63, 255, 256, 257, 511, 512, 513, 1000, 2048, 4096, 4097, 8192,
                                   8193, 10000, 32769, 65537, 131075])
@pytest.mark.parametrize("dtype", TYPES)
def test_vocabularies(vocab, dtype):
    rows = 7 if vocab < 20000 else 3
    x, t = normal(vocab, rows, vocab, dtype=dtype), some(1, rows, vocab)
    check(x, t, top=min(vocab, 20))
    check_grad(x, t, 1.0, normal(2, rows, scale=1.0), normal(3, rows, scale=1.0))


@pytest.mark.parametrize("top", [0, 1, 2, 5, 17, 64, 100, 255, 256])
@pytest.mark.parametrize("vocab", [256, 700, 3001, 20000, 70001])
def test_tops(top, vocab):
    check(normal(top, 4, vocab), some(1, 4, vocab), top=top)


@pytest.mark.parametrize("rows", [1, 2, 5, 100, 256, 700])
def test_rows(rows):
    """One row, cut into parts, to more than run at once."""
    check(normal(rows, rows, 40000 if rows > 5 else 150001, dtype=torch.bfloat16), some(1, rows, 40000), top=9)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [300, 9000, 100003])
def test_ties_go_to_the_lowest_index(dtype, vocab):
    """Few values, one value, zeros of both signs; rows that rise and fall, where no bound from the
    first pieces holds the rest back."""
    rise = torch.arange(vocab, dtype=torch.float32).cuda()
    x = torch.stack([normal(0, vocab).round(), torch.zeros_like(rise), torch.zeros_like(rise), rise / vocab, -rise / vocab,
                     (rise / 1000).floor(), torch.where(rise > vocab - 40, 5.0, 0.0)])
    x[2, ::2] = -0.0
    check(x.to(dtype), some(1, 7, vocab), top=33)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [30, 5000, 70000])
def test_masks(dtype, vocab):
    """Masks of -inf and of the type's lowest value: few places left, one, none, the first pieces shut."""
    low = torch.finfo(dtype).min
    x = normal(0, 10, vocab, dtype=dtype)
    x[0, torch.randperm(vocab, generator=torch.Generator().manual_seed(0)).cuda()[5:]] = -INF
    x[1] = -INF
    x[1, vocab - 1] = 3.0
    x[2] = -INF
    x[3] = low
    x[4, torch.arange(vocab).cuda() % 3 > 0] = low
    x[5, : vocab // 2] = -INF
    x[6, : vocab // 2] = low
    x[7, : vocab // 2] = low
    x[7, vocab // 2:] = -INF
    x[8, vocab // 2:] = low
    t = some(1, 10, vocab)
    t[1], t[5] = vocab - 1, vocab - 2
    check(x, t, top=min(vocab, 12))
    check(x, t, tau=0.3)
    check_grad(x[[0, 1, 3, 4, 5, 6, 7, 8, 9]], t[[0, 1, 3, 4, 5, 6, 7, 8, 9]], 1.0, normal(2, 9, scale=1.0),
               normal(3, 9, scale=1.0))


def test_a_row_of_nothing():
    x, t = torch.full((2, 1000), -INF, device="cuda"), torch.tensor([5, -1]).cuda()
    got = check(x, t, top=3, finite=False)
    assert got.stats.tolist() == [[-INF, -INF]] * 2 and got.entropy.tolist() == [0.0, 0.0]
    assert got.logprob.tolist() == [-INF, 0.0] and got.top_index.tolist() == [[0, 1, 2]] * 2
    one = torch.ones(2, device="cuda")
    assert bool((readout.token_logprobs_grad(x, t, got, one, one) == 0).all())


@pytest.mark.parametrize("vocab", [600, 50000])
def test_logits_far_apart(vocab):
    """The largest logits come late, hundreds above the first; or early."""
    x = normal(0, 4, vocab)
    x[0, -3:] += 300.0
    x[1, :3] += 300.0
    x[2] += torch.linspace(-500.0, 500.0, vocab, device="cuda")
    x[3] -= 1e30
    t = some(1, 4, vocab)
    check(x, t, top=5)
    check(x, t, tau=0.05, top=5)
    check(x, t, tau=50.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_not_finite_stays_in_its_row(dtype):
    for vocab in (40, 3000, 70000):
        x, t = normal(0, 5, vocab, dtype=dtype), some(1, 5, vocab)
        whole = readout.token_logprobs(x, t, top=4)
        x[1, vocab // 2], x[3, 1] = float("nan"), INF
        x[4, -1] = INF
        got = readout.token_logprobs(x, t, top=4)
        hit = [1, 3, 4]
        for a, b in zip(whole, got):
            assert torch.equal(a[[0, 2]], b[[0, 2]])
        for name in ("logprob", "entropy", "top_logprob", "stats"):
            assert bool(getattr(got, name)[hit].isnan().all())
        assert got.top_index[3, 0] == 1 and got.top_index[4, 0] == vocab - 1
        clean = torch.where(x[1].isnan(), -INF, x[1])[None]
        assert torch.equal(got.top_index[1], readout.token_logprobs(clean, t[:1], top=4).top_index[0])
        assert bool(readout.token_logprobs_grad(x, t, got, torch.ones(5, device="cuda"))[hit].isnan().all())


@pytest.mark.parametrize("tau", [1e-30, 0.01, 0.5, 2.0, 1e3, 1e30])
def test_temperatures(tau):
    x, t = normal(0, 6, 2000), some(1, 6, 2000)
    check(x, t, tau=tau, top=6)
    if 0.01 <= tau <= 1e3:
        check_grad(x, t, tau, normal(2, 6, scale=1.0), normal(3, 6, scale=1.0))


def test_sure_answers():
    """Rows whose one place holds nearly all: entropies and gradients of nearly nothing."""
    x = torch.zeros(3, 100, device="cuda")
    x[0, 7], x[1, 7], x[2, 7] = 12.0, 30.0, 200.0
    t = torch.full((3,), 7).cuda()
    check(x, t, top=2)
    check_grad(x, t, 1.0, torch.ones(3, device="cuda"), torch.ones(3, device="cuda"))


def test_tokens_of_every_kind():
    x = normal(0, 5, 77)
    for dtype in (torch.int32, torch.int64):
        t = torch.tensor([0, 76, 77, -1, -100], dtype=dtype).cuda()
        got = check(x, t)
        assert got.logprob[2:].tolist() == [0.0] * 3
        grad = check_grad(x, t, 1.0, torch.ones(5, device="cuda"), None)
        assert bool((grad[2:] == 0).all())
    check(x, torch.tensor([2 ** 40, -2 ** 40, 1, 2, 3]).cuda())


@pytest.mark.parametrize("dtype", TYPES)
def test_views_and_places_of_the_gradient(dtype):
    wide = normal(0, 9, 1003, dtype=dtype)
    x, t = wide[::2, 1:902], some(1, 5, 901)
    check(x, t, top=3)
    pull, turn = normal(2, 5, scale=1.0), normal(3, 5, scale=1.0)
    want = check_grad(x, t, 0.7, pull, turn)
    out = torch.full((5, 1000), 7.0, dtype=dtype, device="cuda")
    check_grad(x, t, 0.7, pull, turn, out=out[:, 50:951])
    assert bool((out[:, :50] == 7.0).all()) and bool((out[:, 951:] == 7.0).all())
    got = readout.token_logprobs(x, t, temperature=0.7)
    kept = wide.clone()
    assert torch.equal(readout.token_logprobs_grad(x, t, got, pull, turn, temperature=0.7, out=x), want)
    assert torch.equal(wide[1::2], kept[1::2]) and torch.equal(wide[:, 902:], kept[:, 902:])
    check(normal(4, 901, 6, dtype=dtype).t(), some(5, 6, 901), top=2)
    check(normal(4, 1, 50, dtype=dtype).expand(4, 50), some(5, 4, 50), top=2)


def test_gradient_against_differences():
    x, t = normal(0, 3, 40, scale=1.0), some(1, 3, 40)
    pull, turn = normal(2, 3, scale=1.0), normal(3, 3, scale=1.0)
    got = readout.token_logprobs_grad(x, t, readout.token_logprobs(x, t, temperature=1.5), pull, turn, temperature=1.5)

    def loss(x):
        _, logprob, entropy, _, _ = definition(x, t, 1.5, 0)
        return float((pull.cpu().double() * logprob + turn.cpu().double() * entropy).sum())

    way = torch.randn(3, 40, generator=torch.Generator().manual_seed(9), dtype=torch.float64)
    wide = x.cpu().double()
    slope = float((got.cpu().double() * way).sum())
    assert abs((loss(wide + 1e-4 * way) - loss(wide - 1e-4 * way)) / 2e-4 - slope) <= 1e-5 * float(
        got.cpu().double().norm() * way.norm())


def test_of_a_drawn_answer():
    """The logarithm that a draw from all places gives is the token's here."""
    x = normal(0, 20, 5000, dtype=torch.bfloat16)
    token, logprob = readout.sample(x, torch.rand(20, generator=torch.Generator().manual_seed(0)).cuda(), temperature=0.8)
    same(readout.token_logprobs(x, token, temperature=0.8).logprob, logprob.cpu().double(), size=2.0)


def test_nothing_to_do():
    got = readout.token_logprobs(torch.empty(0, 9, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), top=2)
    assert [tuple(t.shape) for t in got] == [(0,), (0,), (0, 2), (0, 2), (0, 2)]


@pytest.mark.parametrize("rows,vocab", [(1, 140000), (60, 300), (3, 20000)])
def test_captured(rows, vocab):
    x, t, pull = normal(0, rows, vocab), some(1, rows, vocab), normal(2, rows, scale=1.0)

    def call():
        got = readout.token_logprobs(x, t, top=7)
        return [*got, readout.token_logprobs_grad(x, t, got, pull, pull)]

    captured(call, lambda gen: (x.copy_(torch.randn(rows, vocab, generator=gen).round(decimals=2)),
                                t.copy_(torch.randint(0, vocab, (rows,), generator=gen))))


def test_streams_of_their_own():
    x, t = normal(0, 1, 200000), some(1, 1, 200000)
    want = readout.token_logprobs(x, t, top=5)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            got.append(readout.token_logprobs(x, t, top=5))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(want, g))


def test_refusals():
    x, t = normal(0, 4, 50), some(1, 4, 50)
    got = readout.token_logprobs(x, t)
    pull = torch.ones(4, device="cuda")
    call, grad = readout.token_logprobs, readout.token_logprobs_grad
    for f, error, text in (
            (lambda: call(x[0], t), ValueError, "rows, vocab"),
            (lambda: call(x, t[:3]), ValueError, "tokens has shape"),
            (lambda: call(x, t.float()), TypeError, "tokens is"),
            (lambda: call(x, [1, 2, 3, 4]), TypeError, "tensor"),
            (lambda: call(x, t.cpu()), ValueError, "GPU"),
            (lambda: call(x.double(), t), TypeError, "not float32"),
            (lambda: call(x, t, top=51), HelioxError, "top"),
            (lambda: call(x, t, top=-1), HelioxError, "top"),
            (lambda: call(normal(0, 1, 300), t[:1], top=257), HelioxError, "top"),
            (lambda: call(x, t, top=1.0), TypeError, "whole number"),
            (lambda: call(x, t, temperature=0.0), HelioxError, "temperature"),
            (lambda: call(x, t, temperature=float("nan")), HelioxError, "temperature"),
            (lambda: call(x[:, :0], t), HelioxError, "vocab"),
            (lambda: call(x.clone().requires_grad_(), t), ValueError, "records no graph"),
            (lambda: grad(x, t, tuple(got), pull), TypeError, "token_logprobs"),
            (lambda: grad(x[:3], t[:3], got, pull[:3]), ValueError, "entropy has shape"),
            (lambda: grad(x, t, got, pull.double()), TypeError, "dlogprob is"),
            (lambda: grad(x, t, got, pull, pull[:2]), ValueError, "dentropy has shape"),
            (lambda: grad(x, t, got, pull, out=x.half()), ValueError, "out has to be"),
            (lambda: grad(x[:, :49], t, got, pull, out=x[:, 1:]), HelioxError, "overlaps")):
        with pytest.raises(error, match=text):
            f()
