"""Linear attention with decays on the GPU against the recurrence in 64 bits: outputs, end
states, every gradient and the single step, over types, head layouts, lengths, strides and
decays."""
import pytest
import torch

import readout_util as ref
from heliox_amd import readout

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]

# Bounds on the 2-norm of the error, relative.  Outputs of 16 bits: the result, the masked
# products and the state as it enters a product are each rounded once, at most one unit of the
# type each.  fp32 results (and states, whatever the inputs): sums of up to 2^17 terms whose
# roundings are independent, sqrt(2^17) units.
def bound(dtype):
    return 3 * ref.UNIT[dtype] if dtype != torch.float32 else 2 ** 8.5 * ref.UNIT[torch.float32]


def make(seed, dtype, batch, time, heads, qh, kh, vh, dk, dv, layout="packed"):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    if layout == "packed":
        one = r(batch, time, qh * dk + kh * dk + vh * dv).to(dtype).cuda()
        q, k, v = (x.unflatten(-1, (n, -1)) for x, n in zip(one.split([qh * dk, kh * dk, vh * dv], -1), (qh, kh, vh)))
    elif layout == "heads_first":
        q, k, v = (r(batch, n, time, d).to(dtype).cuda().transpose(1, 2) for n, d in ((qh, dk), (kh, dk), (vh, dv)))
    elif layout == "odd":        # one element past an aligned address, rows of an odd stride
        q, k, v = (r(batch, time, n, d + 3).to(dtype).cuda()[..., 1:d + 1] for n, d in ((qh, dk), (kh, dk), (vh, dv)))
    elif layout == "channels_apart":
        q, k, v = (r(batch, time, d, n).to(dtype).cuda().transpose(2, 3) for n, d in ((qh, dk), (kh, dk), (vh, dv)))
    elif layout == "broadcast":
        q, k, v = (r(1, time, n, d).to(dtype).cuda().expand(batch, -1, -1, -1)
                   for n, d in ((qh, dk), (kh, dk), (vh, dv)))
    # decays from none at all to no memory
    g = torch.tensor([0.0, -0.002, -0.05, -0.4, -3.0, -float("inf"), -0.01, -1e-5])[torch.arange(heads) % 8].cuda()
    state = r(batch, heads, dk, dv).cuda()
    do = r(batch, time, heads, dv).to(dtype).cuda()
    dend = r(batch, heads, dk, dv).cuda()
    return q, k, v, g, state, do, dend


def check(dtype, shape, layout="packed", with_state=True, lengths=None, scale=None, seed=0):
    batch, time, heads, qh, kh, vh, dk, dv = shape
    q, k, v, g, state, do, dend = make(seed, dtype, *shape, layout=layout)
    print(f"case attention {dtype} {shape} {layout} state={with_state} lengths={lengths}", flush=True)
    if lengths is not None:
        for i, n in enumerate(lengths):     # what lies past a length is never looked at
            if layout != "broadcast":
                for x in (q, k, v, do):
                    x[i, n:] = float("nan")
        lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if not with_state:
        state = dend = None
    o, end = readout.linear_attention(q, k, v, g, scale=scale, initial_state=state, lengths=lengths)
    got = readout.linear_attention_grad(q, k, v, g, do, scale=scale, initial_state=state, lengths=lengths, dstate=dend)
    torch.cuda.synchronize()
    want = ref.attention(q, k, v, g, dk ** -0.5 if scale is None else scale, state, lengths, do, dend)
    assert o.dtype == dtype and end.dtype == torch.float32
    assert ref.rel(o, want[0]) <= bound(dtype)
    assert ref.rel(end, want[1]) <= bound(torch.float32)
    for x, w, like in zip(got[:3], want[2:5], (q, k, v)):
        assert x.dtype == dtype and x.shape == like.shape
        assert ref.rel(x, w) <= bound(dtype)
    if with_state:
        assert ref.rel(got[3], want[5]) <= bound(torch.float32)
    else:
        assert got[3] is None
    if lengths is not None:
        for i, n in enumerate(lengths.tolist()):
            assert not o[i, n:].any() and not any(x[i, n:].any() for x in got[:3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("time", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200])
def test_lengths(dtype, time):
    check(dtype, (2, time, 2, 2, 2, 2, 32, 32), seed=time)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dk,dv", [(1, 1), (1, 40), (7, 5), (16, 16), (64, 64), (40, 80), (80, 40), (96, 96), (128, 128),
                                   (129, 17), (200, 130), (160, 256), (256, 256)])
def test_head_sizes(dtype, dk, dv):
    check(dtype, (1, 150, 3, 3, 3, 3, dk, dv), seed=dk + dv)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [(4, 4, 1, 4), (4, 4, 2, 2), (6, 2, 3, 1), (8, 1, 1, 8), (12, 12, 4, 12), (5, 5, 5, 1)])
def test_shared_heads(dtype, heads):
    check(dtype, (2, 90, *heads, 24, 40), seed=sum(heads))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["heads_first", "odd", "channels_apart", "broadcast"])
def test_strides(dtype, layout):
    check(dtype, (3, 77, 2, 2, 1, 2, 33, 48), layout=layout, seed=5)
    check(dtype, (2, 130, 2, 2, 2, 2, 64, 64), layout=layout, seed=6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_state", [True, False])
def test_ragged(dtype, with_state):
    check(dtype, (7, 140, 3, 3, 3, 3, 48, 20), with_state=with_state, lengths=[140, 0, 1, 64, 65, 128, 99], seed=7)


@pytest.mark.parametrize("dtype", TYPES)
def test_long_and_few(dtype):
    """One sequence, one head: the time axis is what fills the chip."""
    check(dtype, (1, 5000, 1, 1, 1, 1, 64, 48), seed=8)
    check(dtype, (2, 3001, 2, 2, 1, 2, 20, 36), lengths=[3001, 1500], seed=9)


@pytest.mark.parametrize("dtype", TYPES)
def test_scale_and_no_state(dtype):
    check(dtype, (2, 70, 8, 8, 8, 8, 32, 64), with_state=False, scale=0.37, seed=10)


def test_empty():
    for batch, time in ((0, 5), (3, 0)):
        q, k, v, g, state, do, dend = make(1, torch.float32, batch, time, 2, 2, 2, 2, 8, 8)
        o, end = readout.linear_attention(q, k, v, g, initial_state=state)
        got = readout.linear_attention_grad(q, k, v, g, do, initial_state=state, dstate=dend)
        assert o.shape == v.shape and torch.equal(end, state) and torch.equal(got[3], dend)
        _, end = readout.linear_attention(q, k, v, g)
        assert not end.any()


def test_large_values_stay_finite():
    """fp16 inputs whose products and states pass fp16's largest number."""
    q, k, v, g, *_ = make(3, torch.float16, 1, 130, 2, 2, 2, 2, 64, 64)
    g = torch.full((2,), -0.003, device="cuda")
    k, q = k * 60, q * 60
    o, end = readout.linear_attention(q, k, v, g, scale=1e-4)
    want = ref.attention(q, k, v, g, 1e-4)
    assert float(want[1].abs().max()) > 400
    assert float((q[0, 0, 0].double() @ k[0, 0, 0].double()).abs()) >= 0
    assert ref.rel(o, want[0]) <= bound(torch.float16) and ref.rel(end, want[1]) <= bound(torch.float32)
    k2 = k * 100
    _, end = readout.linear_attention(q, k2, v * 20, g, scale=1e-9)
    want = ref.attention(q, k2, v * 20, g, 1e-9)
    assert float(want[1].abs().max()) > 65504
    o, _ = readout.linear_attention(q, k2, v * 20, g, scale=1e-7)
    assert ref.rel(end, want[1]) <= bound(torch.float32)
    assert ref.rel(o, want[0] * 100) <= bound(torch.float16)


def test_gradient_against_differences():
    """The loss is linear in each of q, k, v and the initial state, so central differences have
    no error of their own: what is left is the rounding of two losses, each a sum of 2^13
    products good to 2^8.5 units, over the step."""
    shape = (2, 70, 2, 2, 1, 2, 24, 16)
    q, k, v, g, state, do, dend = make(11, torch.float32, *shape)
    g = torch.tensor([-0.02, -0.3], device="cuda")

    def loss(q, k, v, state):
        o, end = readout.linear_attention(q, k, v, g, initial_state=state)
        return (o.double() * do.double()).sum() + (end.double() * dend.double()).sum(), \
            (o.double() * do.double()).norm() + (end.double() * dend.double()).norm()

    grads = readout.linear_attention_grad(q, k, v, g, do, initial_state=state, dstate=dend)
    args = [q, k, v, state]
    for n, grad in enumerate(grads):
        way = torch.randn(args[n].shape, generator=torch.Generator().manual_seed(n)).cuda()
        step = 0.5
        up, down = list(args), list(args)
        up[n], down[n] = args[n] + step * way, args[n] - step * way
        (a, na), (b, nb) = loss(*up), loss(*down)
        diff = float(a - b) / (2 * step)
        exact = float((grad.double() * way.double()).sum())
        assert abs(diff - exact) <= 2 ** 8.5 * ref.UNIT[torch.float32] * float(na + nb) / step


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 1, 1), (3, 4, 4, 4, 4, 64, 64), (5, 6, 6, 2, 3, 40, 33),
                                   (2, 3, 1, 1, 3, 128, 128), (4, 2, 2, 2, 2, 7, 256), (2, 2, 2, 2, 2, 256, 200)])
def test_step(dtype, shape):
    batch, heads, qh, kh, vh, dk, dv = shape
    q, k, v, g, *_ = make(13, dtype, batch, 3, heads, qh, kh, vh, dk, dv)
    pool = torch.randn(batch + 4, heads, dk, dv, generator=torch.Generator().manual_seed(3)).cuda()
    slots = torch.randperm(batch + 4, generator=torch.Generator().manual_seed(4))[:batch].to(torch.int32)
    if batch > 2:
        slots[1], slots[2] = -1, batch + 4      # neither is a slot
    before = pool.clone()
    run = [i for i in range(batch) if 0 <= slots[i] < batch + 4]
    at = slots[run].long().cuda()
    outs = [readout.linear_attention_step(q[:, t], k[:, t], v[:, t], g, pool, slots=slots.cuda()) for t in range(3)]
    o = torch.stack(outs, 1)
    want, end = ref.attention(q[run], k[run], v[run], g, dk ** -0.5, before[at])
    assert o.dtype == dtype and ref.rel(o[run], want) <= bound(dtype)
    assert ref.rel(pool[at], end) <= bound(torch.float32)
    others = torch.ones(batch + 4, dtype=torch.bool, device="cuda")
    others[at] = False
    assert torch.equal(pool[others], before[others])
    assert not o[[i for i in range(batch) if i not in run]].any()


def test_step_goes_on_from_a_recording():
    """Steps after a chunked pass give what the chunked pass over all of it gives."""
    q, k, v, g, *_ = make(17, torch.float32, 2, 101, 3, 3, 3, 3, 32, 48)
    whole, end = readout.linear_attention(q, k, v, g)
    _, state = readout.linear_attention(q[:, :90], k[:, :90], v[:, :90], g)
    for t in range(90, 101):
        o = readout.linear_attention_step(q[:, t], k[:, t], v[:, t], g, state)
        assert ref.rel(o, whole[:, t].cpu().double()) <= 2 * bound(torch.float32)
    assert ref.rel(state, end.cpu().double()) <= 2 * bound(torch.float32)


def test_same_bits_every_time_and_on_another_stream():
    q, k, v, g, state, do, dend = make(19, torch.bfloat16, 2, 700, 4, 4, 2, 1, 64, 64)
    one = [*readout.linear_attention(q, k, v, g, initial_state=state),
           *readout.linear_attention_grad(q, k, v, g, do, initial_state=state, dstate=dend)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two = [*readout.linear_attention(q, k, v, g, initial_state=state),
               *readout.linear_attention_grad(q, k, v, g, do, initial_state=state, dstate=dend)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_captured_into_a_graph():
    q, k, v, g, state, *_ = make(23, torch.bfloat16, 2, 300, 2, 2, 2, 2, 64, 64)
    pool = state.clone()

    def work():
        o, end = readout.linear_attention(q, k, v, g, initial_state=state)
        return o, end, readout.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, pool)

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for n in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(n)).to(q.dtype))
        pool.copy_(state)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [x.clone() for x in got]
        pool.copy_(state)
        want = work()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, want)), n


def test_python_refuses_what_does_not_fit():
    q, k, v, g, state, do, dend = make(29, torch.bfloat16, 2, 9, 4, 4, 2, 4, 16, 24)
    bad = [
        (ValueError, lambda: readout.linear_attention(q, k[:, :8], v, g)),
        (ValueError, lambda: readout.linear_attention(q, k[..., :15], v, g)),
        (ValueError, lambda: readout.linear_attention(q[0], k[0], v[0], g)),
        (TypeError, lambda: readout.linear_attention(q, k.half(), v, g)),
        (TypeError, lambda: readout.linear_attention(q.double(), k.double(), v.double(), g)),
        (TypeError, lambda: readout.linear_attention(q, k, v, g.double())),
        (TypeError, lambda: readout.linear_attention(q, k, v, None)),
        (ValueError, lambda: readout.linear_attention(q, k, v, g.cpu())),
        (ValueError, lambda: readout.linear_attention(q, k, v, g, initial_state=state[:1])),
        (TypeError, lambda: readout.linear_attention(q, k, v, g, lengths=torch.tensor([1, 2], device="cuda"))),
        (ValueError, lambda: readout.linear_attention_grad(q, k, v, g, do[..., :23])),
        (TypeError, lambda: readout.linear_attention_grad(q, k, v, g, do.float())),
        (TypeError, lambda: readout.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state.transpose(2, 3))),
        (ValueError, lambda: readout.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state[:, :3].contiguous())),
        (RuntimeError, lambda: readout.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state[:1])),
        (RuntimeError, lambda: readout.linear_attention(q, k, v, g[:3])),
        (RuntimeError, lambda: readout.linear_attention(q, k, v, g, scale=float("nan"))),
        (ValueError, lambda: readout.sample(q[:, 0, 0], g)),
        (TypeError, lambda: readout.sample(q[:, 0, 0], g[:2], top_k=g[:2])),
        (ValueError, lambda: readout.distill_loss(q[:, 0, 0], torch.zeros(3, 1, dtype=torch.int32, device="cuda"),
                                                  torch.zeros(3, 1, device="cuda"))),
        (TypeError, lambda: readout.distill_loss(q[:, 0, 0], torch.zeros(2, 1, device="cuda"),
                                                 torch.zeros(2, 1, device="cuda"))),
        (ValueError, lambda: readout.distill_loss_grad(q[:, 0, 0], torch.zeros(2, 1, dtype=torch.int32, device="cuda"),
                                                       torch.zeros(2, 1, device="cuda"), out=q[:, 0, 0].t())),
    ]
    for error, call in bad:
        with pytest.raises(error):
            call()


def test_decays_are_clamped_like_the_recurrence():
    """Very strong decays (and none) in one call, over several chunks and segments."""
    q, k, v, *_ = make(31, torch.float32, 1, 2100, 4, 4, 4, 4, 16, 16)
    g = torch.tensor([-1e30, -200.0, -20.0, 0.0], device="cuda")
    o, end = readout.linear_attention(q, k, v, g)
    want = ref.attention(q, k, v, g, 0.25)
    assert ref.rel(o, want[0]) <= bound(torch.float32) and ref.rel(end, want[1]) <= bound(torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_offsets_past_32_bits(dtype):
    """Sequences 2^31 elements apart, steps 2^24 apart, and a state pool of over 2^31 values."""
    far = 2 ** 31 + 64
    space = torch.empty(far + 40 * 2 ** 24 + 64, dtype=dtype, device="cuda")
    gen = torch.Generator().manual_seed(37)
    q, k, v = (torch.randn(2, 40, 1, 16, generator=gen).to(dtype).cuda() for _ in range(3))
    apart = []
    for n, x in enumerate((q, k, v)):
        y = space.as_strided(x.shape, (far, 2 ** 24, 16, 1), 16 * n)
        y.copy_(x)
        apart.append(y)
    g = torch.tensor([-0.05], device="cuda")
    near, far_ = readout.linear_attention(q, k, v, g), readout.linear_attention(*apart, g)
    assert all(torch.equal(a, b) for a, b in zip(near, far_))
    do = torch.randn(2, 40, 1, 16, generator=gen).to(dtype).cuda()
    near, far_ = readout.linear_attention_grad(q, k, v, g, do), readout.linear_attention_grad(*apart, g, do)
    assert all(torch.equal(a, b) for a, b in zip(near[:3], far_[:3]))
    del space, apart, y
    pool = torch.empty(2 ** 31 // (128 * 128) + 3, 1, 128, 128, device="cuda")
    slots = torch.tensor([pool.shape[0] - 1, 0], dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn(2, 1, 128, generator=gen).to(dtype).cuda() for _ in range(3))
    state = torch.randn(2, 1, 128, 128, generator=gen).cuda()
    pool[slots.long()] = state
    o = readout.linear_attention_step(q, k, v, g, pool, slots=slots)
    assert torch.equal(o, readout.linear_attention_step(q, k, v, g, state))
    assert torch.equal(pool[slots.long()], state)


def by_head(x, dim):
    """(..., heads, ...) as (heads, everything else)."""
    return x.detach().cpu().double().movedim(dim, 0).flatten(1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 100, 8, 64, 64), (2, 600, 4, 128, 128), (1, 300, 8, 96, 80), (1, 200, 4, 256, 100)])
def test_outputs_of_16_bits_are_rounded_once(dtype, shape):
    """Head by head, outputs and gradients are as far from the 64-bit result as that result rounded
    to their type: the products' own terms (2^-17 each, a dozen of them at most) add next to nothing
    to a rounding of 2^-9 or 2^-12."""
    batch, time, heads, dk, dv = shape
    print(f"case rounding {dtype} {shape}", flush=True)
    q, k, v, g, state, do, dend = make(41, dtype, batch, time, heads, heads, heads, heads, dk, dv)
    o, _ = readout.linear_attention(q, k, v, g, initial_state=state)
    got = (o, *readout.linear_attention_grad(q, k, v, g, do, initial_state=state, dstate=dend)[:3])
    want = ref.attention(q, k, v, g, dk ** -0.5, state, None, do, dend)
    for x, w in zip(got, (want[0], *want[2:5])):
        x, least, w = by_head(x, 2), by_head(w.to(dtype), 2), by_head(w, 2)
        off, least = (x - w).norm(dim=1), (least - w).norm(dim=1)
        assert bool((off <= 1.01 * least + 12 * 2.0 ** -17 * w.norm(dim=1)).all()), (off / least).tolist()


@pytest.mark.parametrize("share", [1, 2])
def test_heads_up_to_the_limit(share):
    """2^20 heads: each gives what it gives in a call of its own few.  (heads x heads passes 32 bits from
    46341 heads on.)"""
    heads = 2 ** 20
    print(f"case heads {heads} shared by {share}", flush=True)
    q, k, v, g, state, do, dend = make(43, torch.float32, 1, 3, heads, heads, heads // share, heads, 2, 1)
    o, end = readout.linear_attention(q, k, v, g, initial_state=state)
    grads = readout.linear_attention_grad(q, k, v, g, do, initial_state=state, dstate=dend)
    stepped = state.clone()
    step = readout.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, stepped)
    for first in (0, 40000, 2 ** 19, heads - 16):
        at, few = slice(first, first + 16), slice(first // share, (first + 16) // share)
        own = q[:, :, at], k[:, :, few], v[:, :, at], g[at]
        want = readout.linear_attention(*own, initial_state=state[:, at])
        assert torch.equal(o[:, :, at], want[0]) and torch.equal(end[:, at], want[1])
        want = readout.linear_attention_grad(*own, do[:, :, at], initial_state=state[:, at], dstate=dend[:, at])
        for x, w, part in zip(grads, want, (at, few, at)):
            assert torch.equal(x[:, :, part], w)
        assert torch.equal(grads[3][:, at], want[3])
        one = state[:, at].clone()
        want = readout.linear_attention_step(q[:, 0, at], k[:, 0, few], v[:, 0, at], g[at], one)
        assert torch.equal(step[:, at], want) and torch.equal(stepped[:, at], one)


@pytest.mark.parametrize("dtype", TYPES)
def test_decays_are_the_exponentials(dtype):
    """One input at the first step, seen later: e^{g t}, with decays whose products with whole numbers
    are exact.  What is left are the exponentials' own units: three for each chunk gone through (one
    exponential of at most two units, one product), 16 for the rest."""
    time = 1281
    g = torch.tensor([-1 / 16, -3 / 16, -5 / 16, -13 / 16, -23 / 16, -7 / 8], device="cuda")
    heads = g.shape[0]
    lengths = torch.tensor([1, 2, 33, 50, 64, 65, 97, 129, 256, 300, 511, 800, 1100, 1281], dtype=torch.int32, device="cuda")
    one = torch.ones(1, time, heads, 1, dtype=dtype, device="cuda")
    first = torch.zeros_like(one)
    first[:, 0] = 1
    o, _ = readout.linear_attention(one, first, one, g, scale=1.0)
    batch = lambda x: x.expand(lengths.shape[0], -1, -1, -1)  # noqa: E731
    _, end = readout.linear_attention(batch(one), batch(first), batch(one), g, scale=1.0, lengths=lengths)
    t = torch.arange(time, device="cuda").double()
    courses = [(end[:, :, 0, 0].double(), lengths.double() - 1)]
    if dtype == torch.float32:
        courses.append((o[0, :, :, 0].double(), t))
    for got, ago in courses:
        want = torch.exp(g.double() * ago[:, None])
        bound_ = (3 * ago[:, None] / 32 + 16) * ref.UNIT[torch.float32]
        seen = g.double() * ago[:, None] > -80
        off = (got / want - 1).abs()
        assert bool((off <= bound_)[seen].all()), float((off / bound_)[seen].max())


def check_reach(got, want, dtype, what):
    """Finite where the recurrence is, and as near to it as everywhere; not finite where it is not."""
    got, want = got.detach().cpu().double(), want.double()
    there = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), there), (what, int((torch.isfinite(got) != there).sum()))
    got, want = torch.where(there, got, 0.0), torch.where(there, want, 0.0)
    assert float((got - want).norm()) <= bound(dtype) * float(want.norm()), what


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("shape", [(2, 200, 2, 2, 2, 2, 48, 40), (1, 130, 8, 8, 4, 8, 64, 64), (1, 1500, 1, 1, 1, 1, 33, 100)])
def test_what_is_not_finite_reaches_no_earlier_step(dtype, value, shape):
    """One infinity or NaN in one of q, k, v, do: outputs, states and gradients that the recurrence
    does not bring it to are as without it."""
    batch, time, heads, qh, kh, vh, dk, dv = shape
    print(f"case reach {dtype} {value} {shape}", flush=True)
    for n, step in enumerate((0, 5, 63, 64, time // 2 + 1, time - 1)):
        q, k, v, g, state, do, dend = make(47 + n, dtype, *shape)
        name = ("q", "k", "v", "do")[n % 4]
        x = {"q": q, "k": k, "v": v, "do": do}[name]
        x[0, step, 0, 3] = value
        if n == 4:                       # two in one chunk
            v[0, step + 3, 0, 1] = value
        o, end = readout.linear_attention(q, k, v, g, initial_state=state)
        grads = readout.linear_attention_grad(q, k, v, g, do, initial_state=state, dstate=dend)
        want = ref.attention(q, k, v, g, dk ** -0.5, state, None, do, dend)
        for x, w, kind, part in zip((o, end, *grads), want, (dtype, torch.float32, dtype, dtype, dtype, torch.float32),
                                    ("o", "end", "dq", "dk", "dv", "dinitial")):
            check_reach(x, w, kind, (name, step, part))


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_but_nan_ends(dtype):
    """Every step is a chunk of its own then."""
    q, k, v, g, state, *_ = make(59, dtype, 2, 300, 2, 2, 2, 2, 32, 64)
    v[0] = float("nan")
    o, end = readout.linear_attention(q, k, v, g, initial_state=state)
    want = ref.attention(q, k, v, g, 32 ** -0.5, state)
    check_reach(o, want[0], dtype, "o")
    check_reach(end, want[1], torch.float32, "end")


def test_gradients_are_not_lost_in_silence():
    """While torch records, inputs that require a gradient are refused; under no_grad they are not."""
    q, k, v, g, state, do, dend = make(61, torch.float32, 1, 9, 2, 2, 2, 2, 8, 8)
    x, index, t = q[0, :, 0], torch.zeros(9, 1, dtype=torch.int32, device="cuda"), torch.zeros(9, 1, device="cuda")
    lse = torch.ones(9, device="cuda")

    def calls(q=q, k=k, v=v, g=g, state=state, x=x, t=t, lse=lse):
        return {"attention": lambda: readout.linear_attention(q, k, v, g, initial_state=state),
                "step": lambda: readout.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state),
                "distill": lambda: readout.distill_loss(x, index, t, teacher_lse=lse)}

    asks = lambda y: y.clone().requires_grad_()  # noqa: E731
    for names, given in ((("attention", "step"), {"q": asks(q)}), (("attention", "step"), {"k": asks(k)}),
                         (("attention", "step"), {"v": asks(v)}), (("attention", "step"), {"g": asks(g)}),
                         (("attention", "step"), {"state": asks(state)}), (("distill",), {"x": asks(x)}),
                         (("distill",), {"t": asks(t)}), (("distill",), {"lse": asks(lse)})):
        for name in names:
            with pytest.raises(ValueError, match="_grad"):
                calls(**given)[name]()
            with torch.no_grad():
                calls(**given)[name]()
    # the calls that make gradients take what their gradients are for
    readout.linear_attention_grad(asks(q), asks(k), asks(v), g, do, initial_state=asks(state))
    readout.distill_loss_grad(asks(x), index, t)
    readout.sample(asks(x), lse * 0.5)


def test_the_pair_of_calls_in_an_autograd_function():
    """As a model whose other parts are torch's would use them."""
    class Attention(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v, g):
            ctx.save_for_backward(q, k, v, g)
            return readout.linear_attention(q, k, v, g)

        @staticmethod
        def backward(ctx, do, dstate):
            q, k, v, g = ctx.saved_tensors
            return (*readout.linear_attention_grad(q, k, v, g, do, dstate=dstate)[:3], None)

    q, k, v, g, state, do, dend = make(67, torch.float32, 2, 70, 4, 4, 2, 4, 16, 24)
    leaves = [y.clone().requires_grad_() for y in (q, k, v)]
    o, end = Attention.apply(*leaves, g)
    torch.autograd.backward([o, end], [do, dend])
    want = readout.linear_attention_grad(q, k, v, g, do, dstate=dend)
    assert all(torch.equal(y.grad, w) for y, w in zip(leaves, want))


def head_bounds(got, want, dtype, dim):
    """Head by head, so that slow heads do not drown fast ones.  16 bits: as far off as the result's own
    rounding, and a dozen terms of 2^-17.  fp32: sums of up to 2^8 terms a chunk and 2^6 chunks whose
    roundings are independent, 2^4 units, and the decays' units, 2^4 more."""
    x, w = by_head(got, dim), by_head(want, dim)
    off, size = (x - w).norm(dim=1), w.norm(dim=1)
    if dtype == torch.float32:
        return off, 2 ** 5 * ref.UNIT[dtype] * size
    return off, 1.01 * (by_head(want.to(dtype), dim) - w).norm(dim=1) + 12 * 2.0 ** -17 * size


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,lengths", [
    ((1, 900, 4, 4, 4, 4, 128, 128), None), ((2, 700, 3, 3, 1, 3, 96, 80), [700, 333]),
    ((1, 800, 2, 2, 2, 2, 256, 256), None), ((2, 1100, 2, 2, 2, 2, 33, 47), [1100, 20]),
    ((1, 1600, 4, 4, 4, 4, 64, 64), None), ((2, 1000, 4, 4, 4, 4, 64, 64), [400, 1000]),
    ((1, 1300, 2, 1, 2, 2, 47, 33), [900]), ((1, 800, 2, 2, 2, 2, 160, 200), [500])])
def test_segments_of_every_cut(dtype, shape, lengths):
    """Recordings long enough to be cut into segments, at head sizes of each way to lay them out."""
    batch, time, heads, qh, kh, vh, dk, dv = shape
    print(f"case segments {dtype} {shape} {lengths}", flush=True)
    q, k, v, g, state, do, dend = make(71, dtype, *shape)
    at = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    o, end = readout.linear_attention(q, k, v, g, initial_state=state, lengths=at)
    got = readout.linear_attention_grad(q, k, v, g, do, initial_state=state, lengths=at, dstate=dend)
    want = ref.attention(q, k, v, g, dk ** -0.5, state, lengths, do, dend)
    kinds = (dtype, torch.float32, dtype, dtype, dtype, torch.float32)
    for x, w, kind, dim, name in zip((o, end, *got), want, kinds, (2, 1, 2, 2, 2, 1), ("o", "end", "dq", "dk", "dv", "d0")):
        off, most = head_bounds(x, w, kind, dim)
        assert bool((off <= most).all()), (name, (off / most).tolist())


def test_products_past_the_largest_fp16():
    """q.k and the state pass 65504, the outputs do not."""
    q, k, v, g, *_ = make(73, torch.float16, 1, 130, 2, 2, 2, 2, 64, 64)
    g = torch.full((2,), -0.003, device="cuda")
    q, k = q * 100, k * 100
    dots = (q.double().transpose(1, 2) @ k.double().transpose(1, 2).transpose(2, 3)).tril()
    assert float(dots.abs().max()) > 3 * 65504
    o, end = readout.linear_attention(q, k, v * 20, g, scale=1e-5)
    want = ref.attention(q, k, v * 20, g, 1e-5)
    assert float(want[1].abs().max()) > 1e4 and float(want[0].abs().max()) < 65504
    off, most = head_bounds(o, want[0], torch.float16, 2)
    assert bool((off <= most).all())
    off, most = head_bounds(end, want[1], torch.float32, 1)
    assert bool((off <= most).all())


def test_gradient_captured_into_a_graph():
    q, k, v, g, state, do, dend = make(79, torch.bfloat16, 1, 900, 4, 4, 2, 4, 64, 48)

    def change(gen):
        q.copy_(torch.randn(q.shape, generator=gen).to(q.dtype))
        do.copy_(torch.randn(do.shape, generator=gen).to(do.dtype))

    ref.captured(lambda: readout.linear_attention_grad(q, k, v, g, do, initial_state=state, dstate=dend), change)
