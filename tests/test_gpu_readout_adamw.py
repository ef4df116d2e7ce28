"""The AdamW step over many tensors on the GPU against its formula in 64 bits, and the 8-bit moments."""
import pytest
import torch

from heliox_amd import HelioxError, readout
from readout_util import UNIT

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
F32 = 2.0 ** -24
HOW = dict(lr=0.01, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)
# one element, whole blocks of 256 and broken ones, a workgroup's 4096 and more
SIZES = [1, 3, 255, 256, 257, 1000, 4095, 4096, 4099, 20000]


def tensors(seed, sizes, dtype=torch.float32, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=gen) * scale).to(dtype).cuda() for n in sizes]


def held(state, i):
    """Tensor i's moments as they are held, float64 on the CPU (v itself)."""
    at = slice(state.starts[i], state.starts[i] + state.sizes[i])
    m, v = state.m[at].cpu().double(), state.v[at].cpu().double()
    if state.bits == 8:
        of = torch.arange(at.start, at.stop) // 256
        m, v = m * state.m_scale.cpu().double()[of], (v * state.v_scale.cpu().double()[of]) ** 2
    return m, v


def formula(p, g, m, v, t, lr, betas, eps, weight_decay, grad_scale=1.0):
    g = g.cpu().double() * grad_scale
    m, v = betas[0] * m + (1 - betas[0]) * g, betas[1] * v + (1 - betas[1]) * g * g
    step = m / (1 - betas[0] ** t) / ((v / (1 - betas[1] ** t)).sqrt() + eps)
    return p.cpu().double() * (1 - lr * weight_decay) - lr * step, m, v


def near(got, want, rel, size=None):
    off = (got.cpu().double() - want).abs() - rel * (want.abs() if size is None else size)
    assert float(off.max()) <= 0, float(off.max())


def check_step(params, grads, state, t, how=HOW, decays=None):
    """One step from the state as it is held: m and v take three roundings, the step ten more and two
    instructions of one unit each, in all under 16 halves of a step."""
    before = [held(state, i) for i in range(len(params))]
    old = [p.clone() for p in params]
    readout.adamw_step(params, grads, state, **how)
    torch.cuda.synchronize()
    assert int(state.step) == t
    for i, (p, o, g) in enumerate(zip(params, old, grads)):
        here = {**how, "weight_decay": decays[i] if decays else how["weight_decay"]}
        want, m, v = formula(o, g, *before[i], t, **here)
        # beta m and (1 - beta) g may nearly cancel
        size = before[i][0].abs() + g.cpu().double().abs() * here.get("grad_scale", 1.0)
        moved = 16 * F32 * here["lr"] * ((want - o.cpu().double()).abs() / here["lr"] + size / ((v / (1 - here["betas"][1] ** t)).sqrt()
                                                                                              + here["eps"]))
        near(p, want, 1.0, (UNIT[p.dtype] + 8 * F32) * want.abs() + moved + (2.0 ** -25 if p.dtype == torch.float16 else 0.0))
        got_m, got_v = held(state, i)
        if state.bits == 32:
            near(got_m, m, 8 * F32, size)
            near(got_v, v, 8 * F32)
        else:
            # half a step of e4m3 is 2^-4 of a number, 2^-10 of the least ones; in units of the block's
            # largest over 448.  v's root is held, and at least the least number where it is not zero.
            for got, want, root in ((got_m, m, False), (got_v.sqrt(), v.sqrt(), True)):
                blocks = torch.nn.functional.pad(want.abs(), (0, -want.numel() % 256)).view(-1, 256).amax(1)
                unit = (blocks / 448).repeat_interleave(256)[:want.numel()]
                least = 2.0 ** -9 if root else 2.0 ** -10
                bound = torch.maximum(2.0 ** -4 * want.abs(), least * unit) + 16 * F32 * (want.abs() + (0 if root else size))
                near(got, want, 1.0, bound)
                scale = (state.v_scale if root else state.m_scale)[state.starts[i] // 256:][:blocks.numel()]
                near(scale, blocks / 448, 16 * F32, blocks / 448 + (0 if root else float(size.max()) / 448))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", TYPES)
def test_steps(bits, dtype, kind):
    params = tensors(0, SIZES, dtype)
    state = readout.adamw_state(params, bits=bits)
    for t in range(1, 5):
        check_step(params, tensors(t, SIZES, kind), state, t)
    whole = torch.ones(state.m.numel(), dtype=torch.bool)
    for at, n in zip(state.starts, state.sizes):
        whole[at:at + n] = False
    assert bool((state.m.cpu().float()[whole] == 0).all()) and bool((state.v.cpu().float()[whole] == 0).all())


@pytest.mark.parametrize("bits", [8, 32])
def test_many_tensors_of_mixed_types(bits):
    """More than a launch lists, empty ones among them, matrices, decays of their own."""
    shapes = [(n % 7, n) for n in range(1, 150)] + [(300, 20), (5000,)]
    gen = torch.Generator().manual_seed(0)
    params = [torch.randn(s, generator=gen).to(TYPES[i % 3]).cuda() for i, s in enumerate(shapes)]
    grads = [torch.randn(s, generator=gen).to(TYPES[i // 3 % 3]).cuda() for i, s in enumerate(shapes)]
    decays = [0.1 * (i % 4) for i in range(len(shapes))]
    state = readout.adamw_state(params, bits=bits)
    keep = [i for i, p in enumerate(params) if p.numel()]
    old, t = [p.clone() for p in params], 1
    readout.adamw_step(params, grads, state, **{**HOW, "weight_decay": decays})
    for i in keep:
        p, g = old[i].flatten(), grads[i].flatten()
        zero = torch.zeros(p.numel(), dtype=torch.float64)
        want, m, v = formula(p, g, zero, zero, t, **{**HOW, "weight_decay": decays[i]})
        near(params[i].flatten(), want, 1.0, (UNIT[p.dtype] + 8 * F32) * want.abs() + 64 * F32 * HOW["lr"])
        if bits == 32:
            near(held(state, i)[0], m, 8 * F32)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_gradient_that_is_missing(bits):
    params, grads = tensors(0, [300, 500, 40]), tensors(1, [300, 500, 40])
    state = readout.adamw_state(params, bits=bits)
    readout.adamw_step(params, grads, state, **HOW)
    kept, m = params[1].clone(), held(state, 1)
    readout.adamw_step(params, [grads[0], None, grads[2]], state, **HOW)
    assert torch.equal(params[1], kept) and all(torch.equal(a, b) for a, b in zip(m, held(state, 1)))
    assert int(state.step) == 2
    check_step(params[:], grads, state, 3)


def test_settings_on_the_gpu():
    """A learning rate and a clipped norm's factor as tensors give what the numbers give."""
    a, b, grads = tensors(0, SIZES), tensors(0, SIZES), tensors(1, SIZES)
    sa, sb = readout.adamw_state(a), readout.adamw_state(b)
    readout.adamw_step(a, grads, sa, **{**HOW, "lr": 0.02}, grad_scale=0.25)
    readout.adamw_step(b, grads, sb, **{**HOW, "lr": torch.tensor(0.02).cuda()}, grad_scale=torch.tensor([0.25]).cuda())
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(sa.m, sb.m) and torch.equal(sa.v, sb.v)
    c = tensors(0, SIZES)
    check_step(c, grads, readout.adamw_state(c), 1, {**HOW, "grad_scale": 0.25})


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_count_on(bits):
    """Replays with other gradients, rates and scales give what the same steps give one by one."""
    sizes = [700, 5000, 3]
    a, b = tensors(0, sizes), tensors(0, sizes)
    sa, sb = readout.adamw_state(a, bits=bits), readout.adamw_state(b, bits=bits)
    grads, lr, clip = tensors(1, sizes), torch.tensor(0.01).cuda(), torch.ones(1).cuda()

    def step(p, s):
        readout.adamw_step(p, grads, s, **{**HOW, "lr": lr}, grad_scale=clip)

    step(a, sa), step(b, sb)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a, sa)
    for n in range(4):
        for g, new in zip(grads, tensors(10 + n, sizes)):
            g.copy_(new)
        lr.fill_(0.01 * (n + 1)), clip.fill_(1.0 / (n + 1))
        graph.replay()
        torch.cuda.synchronize()
        step(b, sb)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and int(sa.step) == int(sb.step) == n + 2
        assert torch.equal(sa.m.view(torch.uint8), sb.m.view(torch.uint8))
        assert torch.equal(sa.v.view(torch.uint8), sb.v.view(torch.uint8))


def test_parameters_at_odd_addresses():
    for dtype in TYPES:
        flat = tensors(0, [3000], dtype)[0]
        kept = flat.clone()
        params = [flat[1:300], flat[301:1500], flat[1501:2999]]
        grads = [g[1:] for g in tensors(1, [p.numel() + 1 for p in params], dtype)]
        check_step(params, grads, readout.adamw_state(params, bits=8), 1)
        assert torch.equal(flat[[0, 300, 1500, 2999]], kept[[0, 300, 1500, 2999]])
    params = tensors(2, [300])
    view = torch.randn(300, 2, generator=torch.Generator().manual_seed(0)).cuda()[:, 0]
    check_step(params, [view], readout.adamw_state(params), 1)


def test_small_and_large_moments_in_8_bits():
    """Roots far below a block's largest are held as the least number, so that a step stays bounded;
    blocks of nothing, or of less than 2^-100, stay zero."""
    g = torch.ones(256 * 4)
    g[:256] = torch.logspace(-12, 0, 256)
    g[256:512] = 0.0
    g[512:768] = 1e-36
    g[768:] = torch.where(torch.arange(256) == 5, 1.0, 0.0)
    params, grads = [torch.zeros(1024).cuda()], [g.cuda()]
    state = readout.adamw_state(params, bits=8)
    how = dict(lr=1.0, betas=(0.9, 0.99), eps=0.0001, weight_decay=0.0)
    for _ in range(3):
        readout.adamw_step(params, grads, state, **how)
    v = state.v.cpu().float()
    assert bool((v[:256] >= 2.0 ** -9).all()) and bool((v[256:768] == 0).all())
    assert float(v[773]) == 448.0 and int((v[768:] != 0).sum()) == 1
    assert bool((params[0].abs() <= 3 * 1.01).all()) and bool((params[0][256:512] == 0).all())
    assert bool((state.m_scale[1:3] == 0).all()) and bool((state.v_scale[1:3] == 0).all())


def follow(m, v, ms, vs, g, scale, betas):
    """The 8-bit moments' way in torch's fp32, operation by operation."""
    def held(x, floor):
        x = torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256)
        top = x.abs().amax(1, keepdim=True)
        live = top >= 2.0 ** -100
        r = torch.where(live, x / torch.where(live, top, 1.0) * 448.0, 0.0)
        if floor:
            r = torch.where(r > 0, r.clamp(min=2.0 ** -9), r)
        return r.to(torch.float8_e4m3fn).flatten(), torch.where(live, top * torch.tensor(1.0 / 448.0, device=x.device), 0.0)[:, 0]

    n = g.numel()
    g = g.float() * scale
    wide = lambda code, s: (code.float().view(-1, 256) * s[:, None]).flatten()[:n]  # noqa: E731
    m, v = wide(m, ms), wide(v, vs)
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * (v * v) + (1 - betas[1]) * g * g
    return *held(m, False), *held(v.sqrt(), True)


@pytest.mark.parametrize("kind", TYPES)
def test_codes_follow_fp32_arithmetic_to_the_bit(kind):
    """Ten steps of 2 million elements: any other rounding on the way would turn some codes, and these the
    scales of later steps."""
    n = 2_000_001
    params, gen = [torch.zeros(n, device="cuda")], torch.Generator(device="cuda").manual_seed(0)
    state, scale = readout.adamw_state(params, bits=8), torch.tensor([0.7], device="cuda")
    size = torch.exp(torch.randn(n, generator=gen, device="cuda")) * 1e-3
    m, v, ms, vs = (x.clone() for x in (state.m, state.v, state.m_scale, state.v_scale))
    for _ in range(10):
        g = (size * torch.randn(n, generator=gen, device="cuda")).to(kind)
        m, ms, v, vs = follow(m, v, ms, vs, g, scale, (0.9, 0.999))
        readout.adamw_step(params, [g], state, lr=1e-3, grad_scale=scale)
        assert torch.equal(state.m.view(torch.uint8), m.view(torch.uint8))
        assert torch.equal(state.v.view(torch.uint8), v.view(torch.uint8))
        assert torch.equal(state.m_scale, ms) and torch.equal(state.v_scale, vs)


@pytest.mark.parametrize("bits", [8, 32])
def test_what_is_not_finite(bits):
    """It reaches its element, in 8 bits no further than its 256."""
    params, grads = tensors(0, [2000]), tensors(1, [2000])
    clean = [p.clone() for p in params]
    state, other = readout.adamw_state(params, bits=bits), readout.adamw_state(clean, bits=bits)
    for t in range(3):
        bad = [g.clone() for g in grads]
        bad[0][700], bad[0][1300] = float("nan"), float("inf")
        readout.adamw_step(params, bad if t == 0 else grads, state, **HOW)
        readout.adamw_step(clean, grads, other, **HOW)
    keep = torch.ones(2000, dtype=torch.bool)
    if bits == 8:
        keep[512:768] = keep[1280:1536] = False
    else:
        keep[700] = keep[1300] = False
    assert torch.equal(params[0][keep.cuda()], clean[0][keep.cuda()])
    assert not bool(torch.isfinite(params[0][[700, 1300]]).any())


def test_states_are_copied():
    params, grads = tensors(0, SIZES), tensors(1, SIZES)
    state = readout.adamw_state(params, bits=8)
    readout.adamw_step(params, grads, state, **HOW)
    again, copy = [p.clone() for p in params], readout.adamw_state(params, bits=8)
    for name in ("m", "v", "m_scale", "v_scale", "step"):
        getattr(copy, name).copy_(getattr(state, name))
    readout.adamw_step(params, grads, state, **HOW)
    readout.adamw_step(again, grads, copy, **HOW)
    assert all(torch.equal(a, b) for a, b in zip(params, again)) and int(copy.step) == 2


def test_a_graph_of_the_old_values_is_refused():
    """The step is in place: a backward pass that would need the old parameter says so."""
    p = torch.ones(4, device="cuda", requires_grad=True)
    y = (p * p).sum()
    readout.adamw_step([p], [torch.ones(4, device="cuda")], readout.adamw_state([p]), **HOW)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


def test_inference_tensors():
    with torch.inference_mode():
        params, grads = tensors(0, SIZES), tensors(1, SIZES)
        check_step(params, grads, readout.adamw_state(params), 1)


def test_on_a_stream_of_its_own():
    a, b, grads = tensors(0, SIZES), tensors(0, SIZES), tensors(1, SIZES)
    sa, sb = readout.adamw_state(a, bits=8), readout.adamw_state(b, bits=8)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(3):
            readout.adamw_step(a, grads, sa, **HOW)
    for _ in range(3):
        readout.adamw_step(b, grads, sb, **HOW)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_refusals():
    p, g = tensors(0, [300, 40]), tensors(1, [300, 40])
    state = readout.adamw_state(p)
    step = readout.adamw_step
    flat = tensors(2, [500])[0]
    both = [flat[:300], flat[200:240]]
    for f, error, text in (
            (lambda: readout.adamw_state(p, bits=16), ValueError, "bits"),
            (lambda: readout.adamw_state([]), ValueError, "no tensors"),
            (lambda: readout.adamw_state([p[0].cpu()]), ValueError, "GPU"),
            (lambda: readout.adamw_state([p[0].double()]), TypeError, "not float32"),
            (lambda: readout.adamw_state([flat[::2]]), ValueError, "contiguous"),
            (lambda: step(p, g, None, lr=0.1), TypeError, "adamw_state"),
            (lambda: step(p[:1], g[:1], state, lr=0.1), ValueError, "do not fit"),
            (lambda: step(p, g[:1], state, lr=0.1), ValueError, "do not fit"),
            (lambda: step(p[::-1], g[::-1], state, lr=0.1), ValueError, "do not fit"),
            (lambda: step(p, [g[0], g[1].cpu()], state, lr=0.1), ValueError, "GPU"),
            (lambda: step(p, [g[0], g[1].double()], state, lr=0.1), TypeError, "not float32"),
            (lambda: step(p, [g[0], g[1].view(4, 10)], state, lr=0.1), ValueError, "parameters. shapes"),
            (lambda: step(p, g, state, lr=float("nan")), HelioxError, "lr"),
            (lambda: step(p, g, state, lr="0.1"), TypeError, "lr"),
            (lambda: step(p, g, state, lr=torch.ones(2).cuda()), ValueError, "lr has to be one"),
            (lambda: step(p, g, state, lr=torch.tensor(0.1)), ValueError, "GPU"),
            (lambda: step(p, g, state, lr=0.1, betas=(1.0, 0.9)), HelioxError, "beta1"),
            (lambda: step(p, g, state, lr=0.1, betas=(0.9, -0.1)), HelioxError, "beta2"),
            (lambda: step(p, g, state, lr=0.1, betas=0.9), TypeError, "betas"),
            (lambda: step(p, g, state, lr=0.1, eps=-1.0), HelioxError, "eps"),
            (lambda: step(p, g, state, lr=0.1, weight_decay=[0.1]), ValueError, "weight_decay"),
            (lambda: step(p, g, state, lr=0.1, weight_decay=float("inf")), HelioxError, "weight_decay"),
            (lambda: step(p, g, state, lr=0.1, grad_scale=float("inf")), HelioxError, "grad_scale"),
            (lambda: step(both, g, state, lr=0.1), HelioxError, "overlap"),
            (lambda: step([p[0], p[0][:40]], g, state, lr=0.1), HelioxError, "overlap"),
            (lambda: step(p, [g[0], p[0][:40]], state, lr=0.1), HelioxError, "overlap"),
            (lambda: step(p, p, state, lr=0.1), HelioxError, "overlap")):
        with pytest.raises(error, match=text):
            f()
    assert int(state.step) == 0
    step(p, [g[0], g[0][:40]], state, lr=0.1)              # gradients may share what they read
