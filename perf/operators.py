"""The readout operators as timed cases, each with its plain form and an independent 64-bit
result.

A case is a dict of plain values; ``kind`` picks the operator:

  attend   linear attention with a decay for each head over whole recordings (or prompts);
  train    the same, forward and backward: outputs, end states and every gradient;
  step     its recurrent form, one time step for a batch of running sequences, the states
           updated in place;
  distill  the loss against a teacher's top logits, with its gradient by the student's;
  sample   an answer drawn from logits with temperature, top-k, top-p and min-p.

Shapes: ``batch`` sequences of ``time`` steps, ``heads`` heads of ``dk`` x ``dv`` state;
``k_heads`` / ``v_heads`` fewer heads that the others share; ``ragged`` sequences end at
lengths of their own; ``state`` whether a sequence goes on from an earlier state; ``rows`` of
``vocab`` logits, ``top`` of them known of the teacher; ``rest`` whether the teacher's mass
beside them is known too.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CHUNK = 64          # time steps that the plain form takes together
MASS = 2.0 ** 40    # what the sampler's largest weight counts


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # closed loop, one running network: its outputs are read once a tick, pure latency
        {"name": "step_one", "kind": "step", "batch": 1, "heads": 8, "k_heads": 8, "v_heads": 8, "dk": 64, "dv": 64,
         "type": "f32", "slots": 1},
        # many sequences answered at once, their states in a pool larger than the batch
        {"name": "step_batch", "kind": "step", "batch": 256, "heads": 16, "k_heads": 16, "v_heads": 16, "dk": 128,
         "dv": 128, "type": "bf16", "slots": 300},
        # a short recording, one sequence
        {"name": "attend_short", "kind": "attend", "batch": 1, "time": 100, "heads": 8, "k_heads": 8, "v_heads": 8,
         "dk": 64, "dv": 64, "type": "bf16", "ragged": False, "state": False},
        # recordings of unequal lengths that go on from earlier ones; odd head sizes, shared keys
        {"name": "attend_ragged", "kind": "attend", "batch": 13, "time": 777, "heads": 12, "k_heads": 4, "v_heads": 12,
         "dk": 96, "dv": 80, "type": "f16", "ragged": True, "state": True},
        # one long recording: few rows, so the time axis has to be split
        {"name": "attend_long", "kind": "attend", "batch": 1, "time": 65536, "heads": 8, "k_heads": 8, "v_heads": 8,
         "dk": 128, "dv": 128, "type": "bf16", "ragged": False, "state": False},
        # training on captured voltages in their own type: learning ticks of a 200 ms run, small heads
        {"name": "train_voltages", "kind": "train", "batch": 6, "time": 500, "heads": 4, "k_heads": 4, "v_heads": 4,
         "dk": 32, "dv": 32, "type": "f32", "ragged": True, "state": True},
        # training a large readout
        {"name": "train_large", "kind": "train", "batch": 4, "time": 8192, "heads": 16, "k_heads": 16, "v_heads": 16,
         "dk": 128, "dv": 128, "type": "bf16", "ragged": False, "state": False},
        # a classifier of a few hundred classes taught from the five best of its teacher
        {"name": "distill_classes", "kind": "distill", "rows": 100, "vocab": 1000, "top": 5, "type": "f32",
         "rest": False, "temperature": 2.0},
        # odd rows: no row but the first starts at an aligned address, entries absent, the rest's mass known
        {"name": "distill_odd", "kind": "distill", "rows": 517, "vocab": 50021, "top": 33, "type": "f16",
         "rest": True, "temperature": 1.0},
        # a large batch over a large vocabulary
        {"name": "distill_large", "kind": "distill", "rows": 4096, "vocab": 131072, "top": 64, "type": "bf16",
         "rest": True, "temperature": 1.0},
        # one answer: pure latency
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 32000, "type": "bf16"},
        # a batch of answers with settings of their own for each row
        {"name": "sample_batch", "kind": "sample", "rows": 256, "vocab": 131072, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "train", "train", "step", "step", "distill", "distill", "sample", "sample"])
    case = {"kind": kind, "type": rng.choice(["f32", "bf16", "f16"])}
    if kind in ("attend", "train", "step"):
        heads = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
        shared = rng.choice([d for d in (1, 2, 3, 4) if heads % d == 0])
        case |= {"heads": heads, "k_heads": heads // shared, "v_heads": heads // rng.choice([1, shared])}
        for d in ("dk", "dv"):
            case[d] = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128, 160, 256, rng.randint(1, 200)])
        if kind == "step":
            case["batch"] = _log(rng, 1, 256)
            case["slots"] = case["batch"] + rng.randint(0, 30)
            while case["batch"] > 1 and case["batch"] * heads * case["dk"] * case["dv"] > 256 * 16 * 128 * 128:
                case["batch"] //= 2
        else:
            case["batch"] = _log(rng, 1, 32)
            case["time"] = _log(rng, 1, 20000)
            most = (1 << 19 if kind == "attend" else 1 << 18) * 128
            while case["time"] > 1 and case["batch"] * case["time"] * heads * max(case["dk"], case["dv"]) > most:
                case["time"] //= 2
            case |= {"ragged": rng.random() < 0.5, "state": rng.random() < 0.5}
    else:
        case["vocab"] = _log(rng, 2, 131072)
        case["rows"] = _log(rng, 1, 2048)
        while case["rows"] > 1 and case["rows"] * case["vocab"] > (1 << 28 if kind == "distill" else 1 << 25):
            case["rows"] //= 2
        if kind == "distill":
            case |= {"top": min(case["vocab"], _log(rng, 1, 200)), "rest": rng.random() < 0.5,
                     "temperature": rng.choice([0.5, 1.0, 1.0, 2.0, 4.0])}
    return case


# ------------------------------------------------------------------------------ inputs
def _normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    if case["kind"] in ("attend", "train", "step"):
        return {"case": case} | _prepare_attention(case, gen)
    rows, vocab, dtype = case["rows"], case["vocab"], TYPES[case["type"]]
    # a trained model's logits: most of the mass on a small part of the vocabulary
    logits = _normal(gen, rows, vocab, scale=3.0)
    s = {"case": case}
    if case["kind"] == "distill":
        # the teacher agrees with the student in part
        teacher = 0.7 * logits + _normal(gen, rows, vocab, scale=2.0)
        top, index = torch.topk(teacher, case["top"], dim=1)
        # some teachers' rows hold fewer entries than others', some none
        index = torch.where(torch.rand(index.shape, generator=gen, device=DEV) < 0.02, -1, index)
        index[torch.rand(rows, generator=gen, device=DEV) < 0.02] = -1
        s |= {"index": index.to(torch.int32), "teacher": top.to(dtype), "rest": None}
        # the mean over the rows, each with its own weight; in f16 scaled up so that gradients keep their bits
        s["weight"] = torch.rand(rows, generator=gen, device=DEV) * ((1024.0 if case["type"] == "f16" else 1.0) / rows)
        if case["rest"]:
            s["rest"] = torch.logsumexp(teacher / case["temperature"], dim=1)
    else:
        def one_of(*values):
            at = torch.randint(len(values), (rows,), generator=gen, device=DEV)
            return torch.tensor(values, device=DEV)[at]

        s["u"] = torch.rand(rows, generator=gen, device=DEV)
        s["temperature"] = one_of(0.7, 1.0, 1.0, 1.3, 0.0)
        s["top_k"] = one_of(0, 0, 20, 50, 1000).to(torch.int32)
        s["top_p"] = one_of(1.0, 0.95, 0.9, 0.5)
        s["min_p"] = one_of(0.0, 0.0, 0.02, 0.1)
    s["logits"] = logits.to(dtype)
    return s


def _prepare_attention(case, gen):
    b, h, hk, hv, dk, dv = (case[n] for n in ("batch", "heads", "k_heads", "v_heads", "dk", "dv"))
    dtype = TYPES[case["type"]]
    # time constants from 4 steps to 1024, one for each head
    tau = 4.0 * 256.0 ** (torch.arange(h, device=DEV, dtype=torch.float32) / max(h - 1, 1))
    s = {"log_decay": -1.0 / tau, "state": None, "lengths": None}
    if case["kind"] == "step":
        one = _normal(gen, b, h * dk + hk * dk + hv * dv, dtype=dtype)
        s["q"], s["k"], s["v"] = (x.unflatten(-1, (n, -1)) for x, n in
                                  zip(one.split([h * dk, hk * dk, hv * dv], dim=-1), (h, hk, hv)))
        # the pool has a row more than its slots, which the plain form gives to what has no slot
        s["pool"] = _normal(gen, case["slots"] + 1, h, dk, dv)
        s["state"] = s["pool"][:-1]
        slots = torch.randperm(case["slots"], generator=gen, device=DEV)[:b]
        # a sequence that has ended keeps its place in the batch, without a slot
        if b > 4:
            slots = torch.where(torch.rand(b, generator=gen, device=DEV) < 0.05, -1, slots)
        s["slots"] = slots.to(torch.int32)
        return s
    # queries, keys and values come out of one projection, side by side
    one = _normal(gen, b, case["time"], h * dk + hk * dk + hv * dv, dtype=dtype)
    s["q"], s["k"], s["v"] = (x.unflatten(-1, (n, -1)) for x, n in
                              zip(one.split([h * dk, hk * dk, hv * dv], dim=-1), (h, hk, hv)))
    if case["state"]:
        s["state"] = _normal(gen, b, h, dk, dv)
    if case["ragged"]:
        lengths = torch.randint(0, case["time"] + 1, (b,), generator=gen, device=DEV)
        lengths[0] = case["time"]
        if b > 2:
            lengths[1], lengths[2] = 0, 1
        s["lengths"] = lengths.to(torch.int32)
    if case["kind"] == "train":
        s["do"] = _normal(gen, b, case["time"], h, dv, dtype=dtype)
        s["dstate"] = _normal(gen, b, h, dk, dv) if case["state"] else None
    return s


# --------------------------------------------------------------------------------- run
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from heliox_amd import readout

    kind = s["case"]["kind"]
    if kind == "step":
        o = readout.linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], slots=s["slots"])
        return {"o": o, "state": s["state"]}
    if kind in ("attend", "train"):
        how = {"initial_state": s["state"], "lengths": s["lengths"]}
        o, end = readout.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], **how)
        if kind == "attend":
            return {"o": o, "end": end}
        dq, dk, dv, d0 = readout.linear_attention_grad(s["q"], s["k"], s["v"], s["log_decay"], s["do"],
                                                       dstate=s["dstate"], **how)
        got = {"o": o, "end": end, "dq": dq, "dk": dk, "dv": dv}
        return got if d0 is None else got | {"dinitial": d0}
    if kind == "distill":
        loss, grad = readout.distill_loss_grad(s["logits"], s["index"], s["teacher"], teacher_lse=s["rest"],
                                               temperature=s["case"]["temperature"], weight=s["weight"])
        return {"loss": loss, "grad": grad}
    token, logprob = readout.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                    top_p=s["top_p"], min_p=s["min_p"])
    return {"token": token, "logprob": logprob}


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "step":
        return _plain_step(s)
    if kind in ("attend", "train"):
        return _plain_attention(s)
    return _plain_distill(s) if kind == "distill" else _plain_sample(s)


def _per_head(x, heads):
    """(..., heads, d) in 32 bits from (..., fewer heads, d)."""
    return x.float().repeat_interleave(heads // x.shape[-2], dim=-2)


def _plain_step(s):
    """S <- e^g S + k v^T, o = S^T q / sqrt(dk), on the slots of the sequences that run."""
    h, dk, pool = s["case"]["heads"], s["case"]["dk"], s["pool"]
    q, k, v = (_per_head(s[n], h) for n in ("q", "k", "v"))
    live = s["slots"] >= 0
    at = torch.where(live, s["slots"], s["case"]["slots"]).long()
    new = pool[at] * s["log_decay"].exp()[:, None, None] + k[..., :, None] * v[..., None, :]
    o = (q[..., None, :] @ new)[..., 0, :] * dk ** -0.5
    pool[at] = new
    return {"o": torch.where(live[:, None, None], o, 0.0).to(s["q"].dtype), "state": s["state"]}


def _scan(a, b, c, g):
    """y_t = sum over s <= t of e^{g (t - s)} (a_t . b_s) c_s for (B, H, T, D) arrays: chunks of
    CHUNK steps among themselves as masked products, the chunks before them through a state."""
    t = a.shape[2]
    n = -(-t // CHUNK)
    a, b, c = (torch.nn.functional.pad(x, (0, 0, 0, n * CHUNK - t)).unflatten(2, (n, CHUNK)) for x in (a, b, c))
    i = torch.arange(CHUNK, device=a.device, dtype=torch.float32)
    near = torch.where(i[:, None] >= i, torch.exp(g[:, None, None] * (i[:, None] - i).clamp(min=0)), 0.0)
    y = ((a @ b.transpose(-1, -2)) * near[:, None]) @ c
    if n > 1:
        end = (b * torch.exp(g[:, None] * (CHUNK - 1 - i))[:, None, :, None]).transpose(-1, -2) @ c
        j = torch.arange(n, device=a.device, dtype=torch.float32)
        far = torch.where(j[:, None] > j, torch.exp(g[:, None, None] * CHUNK * (j[:, None] - 1 - j).clamp(min=0)), 0.0)
        before = (far @ end.flatten(-2)).unflatten(-1, end.shape[-2:])
        y = y + torch.exp(g[:, None] * (i + 1))[:, None, :, None] * (a @ before)
    return y.flatten(2, 3)[:, :, :t]


def _plain_attention(s):
    case, g, s0 = s["case"], s["log_decay"], s["state"]
    h, t, dk, kind = case["heads"], case["time"], case["dk"], s["q"].dtype
    scale = dk ** -0.5
    q, k, v = (_per_head(s[n], h).transpose(1, 2) for n in ("q", "k", "v"))
    i = torch.arange(t, device=q.device)
    lengths = s["lengths"].long() if s["lengths"] is not None else torch.full((q.shape[0],), t, device=q.device)
    live = (i < lengths[:, None])[:, None, :, None]
    q, k, v = (torch.where(live, x, 0.0) for x in (q, k, v))
    # what is left at the end of what came in at a step, and of the state from before
    left = torch.exp(g[:, None] * (lengths[:, None, None] - 1 - i).clamp(min=0).float())[..., None]
    whole = torch.exp(g * lengths[:, None].float())[..., None, None]
    since = torch.exp(g[:, None] * (i + 1).float())[..., None]
    o = _scan(q, k, v, g)
    end = (k * left).transpose(-1, -2) @ v
    if s0 is not None:
        o = o + since * (q @ s0)
        end = end + whole * s0

    def back(x, like):
        """(B, H, T, D) as (B, T, heads of `like`, D): what heads share adds up."""
        x = x.transpose(1, 2)
        return x.unflatten(2, (like.shape[2], -1)).sum(3).to(kind)

    got = {"o": back(o * scale, s["q"]), "end": end}
    if case["kind"] == "attend":
        return got
    do = torch.where(live, s["do"].float().transpose(1, 2), 0.0) * scale
    dend = s["dstate"]
    turn = lambda x: x.flip(2)  # noqa: E731
    dq = _scan(do, v, k, g)
    dk_ = turn(_scan(turn(v), turn(do), turn(q), g))
    dv_ = turn(_scan(turn(k), turn(q), turn(do), g))
    if s0 is not None:
        dq = dq + since * (do @ s0.transpose(-1, -2))
        got["dinitial"] = (q * since).transpose(-1, -2) @ do + whole * dend
        dk_ = dk_ + left * (v @ dend.transpose(-1, -2))
        dv_ = dv_ + left * (k @ dend)
    dk_, dv_ = (torch.where(live, x, 0.0) for x in (dk_, dv_))
    return got | {"dq": back(dq, s["q"]), "dk": back(dk_, s["k"]), "dv": back(dv_, s["v"])}


def _plain_distill(s):
    """t^2 KL(teacher | student) over the teacher's entries and, where its mass beside them is
    known, one more class for all the others; its gradient by the student's logits."""
    tau = s["case"]["temperature"]
    x = s["logits"].float() / tau
    here = s["index"] >= 0
    at = s["index"].long().clamp(min=0)
    e = torch.exp(x - x.amax(1, keepdim=True))
    z = e.sum(1, keepdim=True)
    lse = z.log() + x.amax(1, keepdim=True)
    q = e / z
    member = torch.zeros_like(x).scatter_add_(1, at, here.float())
    t = torch.where(here, s["teacher"].float() / tau, -torch.inf)
    if s["rest"] is None:
        top = t.amax(1, keepdim=True)
        w = torch.where(here, torch.exp(t - torch.where(top > -torch.inf, top, 0.0)), 0.0)
        mass = w.sum(1, keepdim=True)
        p = torch.where(mass > 0, w / mass, 0.0)
        logp = t - top - mass.log()
    else:
        logp = t - s["rest"][:, None]
        p = torch.where(here, torch.exp(logp), 0.0)
    logq = x.gather(1, at) - lse
    loss = torch.where(p > 0, p * (logp - logq), 0.0).sum(1)
    inside = others = p.sum(1, keepdim=True)
    if s["rest"] is not None:
        p_rest = (1 - p.sum(1, keepdim=True)).clamp(min=0)
        q_rest = torch.where(member > 0, 0.0, q).sum(1, keepdim=True)
        both = (p_rest > 0) & (q_rest > 0)
        loss = loss + torch.where(both, p_rest * (p_rest.log() - q_rest.log()), 0.0)[:, 0]
        # a row without entries is one class: nothing to learn
        some = here.any(1, keepdim=True)
        inside = torch.where(both & some, inside + p_rest, inside)
        others = torch.where(both & some, inside - p_rest / q_rest, inside)
        loss = torch.where(some[:, 0], loss, 0.0)
    grad = q * torch.where(member > 0, inside, others)
    grad = grad.scatter_add_(1, at, -p)
    return {"loss": loss * tau * tau, "grad": (grad * (tau * s["weight"][:, None])).to(s["logits"].dtype)}


def _plain_sample(s):
    """Weights e^{(x - max) / t} counted in units of 2^-40, so that sums are whole numbers; kept
    are the top_k largest (ties: the lowest index), of those the first whose sum from the top
    reaches top_p of theirs, of those what is at least min_p of the largest; the token is the
    first in index order whose running sum is over u of the kept sum."""
    x = s["logits"].float()
    x = torch.where(x.isnan(), -torch.inf, x)
    top = x.amax(1, keepdim=True)
    greedy = s["temperature"][:, None] <= 0
    cold = torch.where(greedy, 1.0, 1.0 / s["temperature"][:, None])
    z = torch.where(x == top, 0.0, (x - top) * cold)
    e = torch.exp(z)
    mass = (e * MASS).long()
    _, order = torch.sort(x, dim=1, descending=True, stable=True)
    m, rank = mass.gather(1, order), torch.arange(x.shape[1], device=x.device)
    k = torch.where(greedy, 1, s["top_k"][:, None])
    m = torch.where((k <= 0) | (rank < k), m, 0)
    before = m.cumsum(1) - m
    p = s["top_p"][:, None].double()
    kept = (before.double() < p * m.sum(1, keepdim=True).double()) | (p >= 1) | (rank == 0)
    kept &= e.gather(1, order) >= s["min_p"][:, None].clamp(max=1.0)
    m = torch.zeros_like(mass).scatter_(1, order, torch.where(kept, m, 0))
    run_ = m.cumsum(1)
    total = run_[:, -1:]
    r = torch.minimum((s["u"][:, None].double() * total.double()).floor().long(), total - 1)
    token = (run_ <= r).sum(1, keepdim=True)
    logprob = z.gather(1, token) - (total.float() / MASS).log()
    nothing = top == -torch.inf
    token, logprob = torch.where(nothing, -1, token), torch.where(nothing, -torch.inf, logprob)
    return {"token": token[:, 0], "logprob": logprob[:, 0]}


# -------------------------------------------------------------------------------- work
def work(case):
    kind, size = case["kind"], TYPES[case["type"]].itemsize
    if kind in ("attend", "train", "step"):
        h, hk, hv, dk, dv = (case[n] for n in ("heads", "k_heads", "v_heads", "dk", "dv"))
        n = case["batch"] * case.get("time", 1)
        tokens, states = n * size, 4 * case["batch"] * h * dk * dv
        ins, out, cell = h * dk + hk * dk + hv * dv, h * dv, n * h * dk * dv
        # a step's state takes one product and one sum for each of its cells, the output the same
        if kind == "step":
            return {"bytes": tokens * (ins + out) + 2 * states, "flops": 4 * cell}
        held = states * (2 if case["state"] else 1)
        if kind == "attend":
            return {"bytes": tokens * (ins + out) + held, "flops": 4 * cell}
        return {"bytes": tokens * (2 * ins + 2 * out) + held + (2 * states if case["state"] else 0),
                "flops": 14 * cell}
    n = case["rows"] * case["vocab"]
    if kind == "distill":
        return {"bytes": 2 * n * size + case["rows"] * (case["top"] * (4 + size) + 8 + 4 * case["rest"]),
                "flops": 6 * n}
    return {"bytes": n * size + case["rows"] * 32, "flops": 4 * n}


# ------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("attend", "train", "step"):
        return _exact_attention(s)
    return _exact_distill(s) if kind == "distill" else _exact_sample(s)


def _exact_attention(s):
    """The recurrence itself, one step after another."""
    case = s["case"]
    h, scale = case["heads"], 1.0 / math.sqrt(case["dk"])
    wide = lambda x: x.double().repeat_interleave(h // x.shape[-2], dim=-2)  # noqa: E731
    q, k, v = wide(s["q"]), wide(s["k"]), wide(s["v"])
    decay = s["log_decay"].double().exp()[None, :, None, None]
    if case["kind"] == "step":
        state = s["state"].double()
        o = torch.zeros(*q.shape[:2], case["dv"], dtype=torch.float64, device=q.device)
        for i, at in enumerate(s["slots"].tolist()):
            if at >= 0:
                state[at] = state[at] * decay[0] + k[i, :, :, None] * v[i, :, None, :]
                o[i] = scale * torch.einsum("hk,hkv->hv", q[i], state[at])
        return {"o": o, "state": state}
    batch, steps = q.shape[:2]
    shape = (batch, h, case["dk"], case["dv"])
    zeros = torch.zeros(shape, dtype=torch.float64, device=q.device)
    state = s["state"].double().clone() if s["state"] is not None else zeros.clone()
    lengths = s["lengths"] if s["lengths"] is not None else torch.full((batch,), steps, device=q.device)
    live = torch.arange(steps, device=q.device)[None] < lengths[:, None]
    keep = torch.where(live[:, :, None, None, None], decay[:, None], 1.0)
    q, k, v = (torch.where(live[:, :, None, None], x, 0.0) for x in (q, k, v))
    train = case["kind"] == "train"
    do = torch.where(live[:, :, None, None], s["do"].double(), 0.0) * scale if train else None
    o, dq, dk, dv = torch.zeros_like(v), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for t in range(steps):
        state.mul_(keep[:, t]).addcmul_(k[:, t, :, :, None], v[:, t, :, None, :])
        o[:, t] = (q[:, t, :, None, :] @ state)[:, :, 0]
        if train:
            dq[:, t] = (state @ do[:, t, :, :, None])[..., 0]
    share = lambda x, like: x.unflatten(2, (like.shape[2], -1)).sum(3)  # noqa: E731
    got = {"o": o * scale, "end": state}
    if not train:
        return got
    back = s["dstate"].double().clone() if s["dstate"] is not None else zeros.clone()
    for t in reversed(range(steps)):
        back.addcmul_(q[:, t, :, :, None], do[:, t, :, None, :])
        dk[:, t] = (back @ v[:, t, :, :, None])[..., 0]
        dv[:, t] = (k[:, t, :, None, :] @ back)[:, :, 0]
        back.mul_(keep[:, t])
    dk, dv = (torch.where(live[:, :, None, None], x, 0.0) for x in (dk, dv))
    got |= {"dq": share(dq, s["q"]), "dk": share(dk, s["k"]), "dv": share(dv, s["v"])}
    return got | {"dinitial": back} if s["state"] is not None else got


def _exact_distill(s):
    tau = s["case"]["temperature"]
    n, width = s["logits"].shape
    loss = torch.zeros(n, dtype=torch.float64, device=s["logits"].device)
    grad = torch.zeros(n, width, dtype=torch.float64, device=s["logits"].device)
    for lo in range(0, n, 256):
        rows = slice(lo, min(n, lo + 256))
        logq = torch.log_softmax(s["logits"][rows].double() / tau, dim=1)
        entry = s["index"][rows].long()
        there = entry >= 0
        where = torch.where(there, entry, width)
        t = torch.where(there, s["teacher"][rows].double() / tau, -torch.inf)
        t = t - (torch.logsumexp(t, 1, keepdim=True) if s["rest"] is None else s["rest"][rows].double()[:, None])
        some = there.any(1, keepdim=True)
        p = torch.where(there & some, t.exp(), 0.0)
        padded = torch.cat([logq, torch.zeros_like(logq[:, :1])], 1)
        part = torch.where(p > 0, p * (t - padded.gather(1, where)), 0.0).sum(1, keepdim=True)
        inside = torch.zeros_like(padded, dtype=torch.bool).scatter_(1, where, True)[:, :-1]
        q = logq.exp()
        factor = p.sum(1, keepdim=True).expand_as(q)
        if s["rest"] is not None:
            p_rest = 1 - p.sum(1, keepdim=True)
            q_rest = torch.where(inside, 0.0, q).sum(1, keepdim=True)
            known = (p_rest > 0) & (q_rest > 0)
            part = part + torch.where(known, p_rest * torch.log(p_rest / q_rest), 0.0)
            factor = torch.where(known, factor + p_rest, factor)
            factor = torch.where(known & ~inside, factor - p_rest / q_rest, factor)
        full = torch.zeros_like(padded).scatter_add_(1, where, p)[:, :-1]
        loss[rows] = torch.where(some, part, 0.0)[:, 0] * tau * tau
        grad[rows] = torch.where(some, q * factor - full, 0.0) * tau * s["weight"][rows].double()[:, None]
    return {"loss": loss, "grad": grad}


def _exact_sample(s):
    """Row by row in 64 bits; the tokens follow, so only their logarithms are compared."""
    logits = s["logits"].double().cpu()
    settings = [s[n].cpu().tolist() for n in ("u", "temperature", "top_k", "top_p", "min_p")]
    out = []
    for row, u, temp, top_k, top_p, min_p in zip(logits, *settings):
        if temp <= 0:
            out.append(0.0)
            continue
        e = torch.exp((row - row.max()) / temp)
        unit = torch.floor(e * MASS)
        value, order = torch.sort(row, descending=True, stable=True)
        count = top_k if 0 < top_k < row.numel() else row.numel()
        if top_p < 1:
            mass = unit[order[:count]].cumsum(0)
            count = 1 + int((mass[:-1] < top_p * mass[-1]).sum())
        chosen = torch.zeros(row.numel(), dtype=torch.bool)
        chosen[order[:count]] = True
        chosen &= e >= min(min_p, 1.0)
        total = torch.where(chosen, unit, 0.0).cumsum(0)
        token = int(torch.searchsorted(total, math.floor(u * float(total[-1])), right=True))
        out.append(math.log(float(unit[token]) / float(total[-1])))
    return {"token": None, "logprob": torch.tensor(out, dtype=torch.float64, device=s["logits"].device)}
