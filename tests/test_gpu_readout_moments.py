"""AdamW's 8-bit moments over many steps: what their codes are, and that they follow the gradients."""
import pytest
import torch

from heliox_amd import readout

pytestmark = pytest.mark.gpu

ROOT2, ROOT3, ROOT11, ROOT17 = 0x6A09E667, 0xBB67AE85, 0x510E527F, 0x1F83D9AB
WORD = 0xFFFFFFFF


def bits(n, t):
    """Of each element from a start at a multiple of 4 on: (the root's, m's), 16 bits each."""
    h = (torch.arange(-(-n // 4), device="cuda") * ROOT2 + (t * ROOT3 & WORD)) & WORD
    h = ((h ^ h >> 16) * ROOT11) & WORD
    h = ((h ^ h >> 15) * ROOT17) & WORD
    h = h ^ h >> 16
    one = torch.stack([(h << k | h >> 32 - k) & WORD for k in (0, 8, 16, 24)], 1).flatten()[:n]
    return one >> 16, one & 0xFFFF


def held(x, floor, cut):
    """Codes and scales of x; cut: 16 bits for each element, None where codes are rounded to nearest."""
    n = x.numel()
    pad = lambda t: torch.nn.functional.pad(t, (0, -n % 256)).view(-1, 256)  # noqa: E731
    x = pad(x)
    top = x.abs().amax(1, keepdim=True)
    live = top >= 2.0 ** -100
    r = torch.where(live, x / torch.where(live, top, 1.0) * 448.0, 0.0)
    some = r > 0
    if cut is not None:
        # the 20 bits that a code drops; codes of numbers under 2^-6 are 2^-9 apart
        add, size = pad(cut) * 16 + 8, r.abs()
        low = ((size.view(torch.int32).long() + add) & ~0xFFFFF).int().view(torch.float32)
        least = (((size * 2.0 ** 29).long() + add) >> 20) * 2.0 ** -9
        r = torch.copysign(torch.where(size < 2.0 ** -6, least, low), r)
    if floor:
        r = torch.where(some, r.clamp(min=2.0 ** -9), r)
    return r.to(torch.float8_e4m3fn).flatten(), torch.where(live, top * torch.tensor(1.0 / 448.0, device="cuda"), 0.0)[:, 0]


@pytest.mark.parametrize("betas,first", [((0.9, 0.999), 996), ((0.95, 0.9), 17), ((0.9, 0.99), 100_000), ((0.0, 0.0), 0),
                                         ((0.5, 0.75), 2 ** 33)])
def test_codes_to_the_bit(betas, first):
    """Eight steps around the last one that rounds to nearest, and later ones."""
    n = 200_003
    params, gen = [torch.zeros(n, device="cuda")], torch.Generator(device="cuda").manual_seed(0)
    state = readout.adamw_state(params, bits=8)
    state.step.fill_(first)
    size = torch.exp(2 * torch.randn(n, generator=gen, device="cuda")) * 1e-3
    m, v, ms, vs = (x.clone() for x in (state.m, state.v, state.m_scale, state.v_scale))
    wide = lambda code, s: (code.float().view(-1, 256) * s[:, None]).flatten()[:n]  # noqa: E731
    for t in range(first + 1, first + 9):
        g = size * torch.randn(n, generator=gen, device="cuda")
        wm, wv = wide(m, ms), wide(v, vs)
        wm = betas[0] * wm + (1 - betas[0]) * g
        wv = betas[1] * (wv * wv) + (1 - betas[1]) * g * g
        cut_v, cut_m = bits(n, t) if t > round(1 / (1 - max(betas))) else (None, None)
        m, ms = held(wm, False, cut_m)
        v, vs = held(wv.sqrt(), True, cut_v)
        readout.adamw_step(params, [g], state, lr=1e-3, betas=betas)
        assert torch.equal(state.m.view(torch.uint8), m.view(torch.uint8)), t
        assert torch.equal(state.v.view(torch.uint8), v.view(torch.uint8)), t
        assert torch.equal(state.m_scale, ms) and torch.equal(state.v_scale, vs)


def both(n):
    params = [[torch.zeros(n, device="cuda")] for _ in range(2)]
    return params, [readout.adamw_state(p, bits=b) for p, b in zip(params, (8, 32))]


def ratios(x, near, share, within):
    """Within `near` of 1, as a factor, at the first and last hundredth; at most `share` of all beyond `within`."""
    low, mid, high = torch.quantile(x, torch.tensor([0.01, 0.5, 0.99], device="cuda")).tolist()
    assert 1 / near <= low and high <= near and 0.9 <= mid <= 1.1, (low, mid, high)
    assert float(((x > within) | (x < 1 / within)).float().mean()) <= share


def test_roots_follow_gradients_that_change():
    """8000 steps of 16384 gradients whose sizes change places after 3000, against moments in 32 bits.

    A root r moves by about (1 - beta2) / 2 = 0.0005 of itself a step (the mean of |g^2 / v - 1| is 0.97 for normal
    gradients), so that its rounding, codes being u <= 1/8 of it apart, adds a variance of 0.0005 u r^2 at most; the
    moment forgets it at a rate of 0.001 a step: a standard deviation of sqrt(0.0005 / 8 / 0.002) = 0.177 at most, 99%
    within a factor of exp(2.33 * 0.177) = 1.51, and 2 is 3.9 of them away.  While a root falls, it forgets nothing: after
    5000 steps the deviation is sqrt(5000 * 0.0005 * 0.09) = 0.47, 14% are off by 2, and 4% of the elements fall so far
    that they still do (by a factor over 12, of sizes with a logarithm's deviation of 1.41)."""
    n = 16384
    params, (eight, wide) = both(n)
    gen = torch.Generator(device="cuda").manual_seed(0)
    size = torch.exp(torch.randn(n, generator=gen, device="cuda")) * 1e-3
    places = torch.randperm(n, generator=gen, device="cuda")
    for t in range(1, 8001):
        g = [size * torch.randn(n, generator=gen, device="cuda")]
        for p, s in zip(params, (eight, wide)):
            readout.adamw_step(p, g, s, lr=1e-3)
        if t in (3000, 8000):
            root = eight.v.float() * eight.v_scale.repeat_interleave(256)
            ratios(root / wide.v.sqrt(), 1.6 if t == 3000 else 2.0, 1e-3 if t == 3000 else 0.02, 2.0)
        if t == 3000:
            size = size[places]


def test_first_moments_follow_gradients_without_noise():
    """Gradients that are nearly the same each step, with beta1 = 0.95: a moment that is off by up to 1.25 of itself
    moves by 0.05 of that, half a step of its code, and would stand still if it were rounded to nearest.  Each rounding is off by at most u / 2 = 1/16 of the moment, unbiased, and counts
    20 times: the mean of 800 is off by 20 / 16 / sqrt(800) = 0.044 of itself, 99% by 0.103."""
    n = 16384
    params, (eight, wide) = both(n)
    gen = torch.Generator(device="cuda").manual_seed(0)
    size = torch.exp(torch.randn(n, generator=gen, device="cuda")) * 1e-3
    size *= torch.sign(torch.randn(n, generator=gen, device="cuda"))
    places = torch.randperm(n, generator=gen, device="cuda")
    sums = torch.zeros(2, n, device="cuda")
    for t in range(1, 2501):
        if t == 1501:
            size = size[places]
        g = [size * (1 + 0.05 * torch.randn(n, generator=gen, device="cuda"))]
        for p, s in zip(params, (eight, wide)):
            readout.adamw_step(p, g, s, lr=1e-3, betas=(0.95, 0.999))
        if t > 1700:
            sums[0] += eight.m.float() * eight.m_scale.repeat_interleave(256)
            sums[1] += wide.m
    ratios(sums[0] / sums[1], 1.15, 1e-3, 1.25)


def test_late_steps_repeat_and_replay():
    """The same calls give the same state, one by one and captured; other steps round otherwise."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    sizes = [700, 5000, 3]
    start = [torch.randn(n, generator=gen, device="cuda") for n in sizes]
    grads = [torch.randn(n, generator=gen, device="cuda") for n in sizes]
    runs = []
    for first in (2000, 2000, 2001):
        params = [p.clone() for p in start]
        state = readout.adamw_state(params, bits=8)
        state.step.fill_(first)
        runs.append((params, state))
    for params, state in runs:
        readout.adamw_step(params, grads, state, lr=1e-3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        readout.adamw_step(runs[0][0], grads, runs[0][1], lr=1e-3)
    for n in range(3):
        for g in grads:
            g.copy_(torch.randn(g.shape, generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for params, state in runs[1:]:
            readout.adamw_step(params, grads, state, lr=1e-3)
        torch.cuda.synchronize()
        (a, sa), (b, sb), (_, sc) = runs
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and int(sa.step) == int(sb.step)
        for name in ("m", "v"):
            code = [getattr(s, name).view(torch.uint8) for s in (sa, sb, sc)]
            assert torch.equal(code[0], code[1]) and not torch.equal(code[0], code[2])


def test_late_steps_keep_what_is_not_finite_where_it_is():
    """A NaN stays with its element, an infinity reaches its 256; zeros, the filling and roots' least codes stay."""
    n = 1000
    params, gen = [torch.zeros(n, device="cuda")], torch.Generator(device="cuda").manual_seed(0)
    state = readout.adamw_state(params, bits=8)
    state.step.fill_(5000)
    g = torch.randn(n, generator=gen, device="cuda")
    g[:8] = torch.tensor([0.0, -0.0, 1e-12, -1e-12, 1e-3, 5.0, -5.0, 0.0], device="cuda")
    g[300], g[600] = float("nan"), float("inf")
    for _ in range(20):
        readout.adamw_step(params, [g], state, lr=1e-3)
    m, v = state.m.float(), state.v.float()
    assert bool((m[n:] == 0).all()) and bool((v[n:] == 0).all())
    assert float(m[0]) == float(m[1]) == float(v[0]) == float(v[1]) == 0.0 and float(v[2]) == float(v[3]) == 2.0 ** -9
    bad = ~torch.isfinite(params[0])
    assert torch.equal(bad.nonzero()[:, 0][:1].cpu(), torch.tensor([300])) and int(bad[256:512].sum()) == 1
    assert not bool(bad[:256].any()) and not bool(bad[768:].any()) and bool(bad[600])
    assert bool(m[300].isnan()) and int(m[256:512].isnan().sum()) == 1
