"""Operators of a trained recurrent readout as timed cases, each with its plain form and an
independent 64-bit result.

A case is a dict of plain values; ``kind`` picks the operator:

  recur        a gated recurrence over whole recordings: h_t = a_t h_{t-1} + (1 - a_t) x_t with
               a = sigmoid(gate);
  recur_train  the same, forward and backward: outputs, end states and every gradient;
  recur_step   one time step for a batch of running sequences, the states updated in place;
  norm         layer norm over the last dimension;
  norm_train   the same, forward and backward, with the gradients of weight and bias;
  score        log probabilities of given tokens, entropies and the top alternatives;
  score_train  the same, and the gradient of both by the logits;
  adamw        an AdamW step over many tensors at once, states in 32 bits or in 8.

Shapes: ``batch`` sequences of ``time`` steps of ``channels``; ``ragged`` sequences end at
lengths of their own; ``state`` whether a sequence goes on from an earlier state; ``rows`` of
``width`` values or ``vocab`` logits, ``top`` alternatives of each; ``tensors`` of ``elements``
in all.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CHUNK = 64                                  # time steps that the plain recurrence takes together
BLOCK = 256                                 # elements that share a scale in 8-bit states
TOP8, LEAST8 = 448.0, 2.0 ** -9             # of the 8-bit floating type: largest and smallest values
EPS = 1e-5
LR, BETAS, ADAM_EPS = 1e-3, (0.9, 0.999), 1e-8


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # closed loop: one tick of many running networks' readouts, pure latency
        {"name": "recur_step", "kind": "recur_step", "batch": 64, "channels": 1024, "slots": 80, "type": "bf16"},
        # recordings of unequal lengths that go on from earlier ones, odd channels
        {"name": "recur_ragged", "kind": "recur", "batch": 13, "time": 777, "channels": 601, "type": "f16",
         "ragged": True, "state": True},
        # one long recording: few rows, so the time axis has to be split
        {"name": "recur_long", "kind": "recur", "batch": 1, "time": 65536, "channels": 512, "type": "f32",
         "ragged": False, "state": False},
        # training a large readout
        {"name": "recur_train", "kind": "recur_train", "batch": 8, "time": 4096, "channels": 2048, "type": "bf16",
         "ragged": False, "state": True},
        # the voltages of one tick, as they were captured: pure latency
        {"name": "norm_tick", "kind": "norm", "rows": 1, "width": 500, "type": "f32"},
        # recordings of odd width
        {"name": "norm_train_odd", "kind": "norm_train", "rows": 5003, "width": 1001, "type": "f16"},
        # training a large readout
        {"name": "norm_train_large", "kind": "norm_train", "rows": 32768, "width": 4096, "type": "bf16"},
        # one answer looked at with its alternatives
        {"name": "score_one", "kind": "score", "rows": 1, "vocab": 32000, "top": 20, "type": "bf16", "temperature": 1.0},
        # many answers over a large vocabulary
        {"name": "score_batch", "kind": "score", "rows": 2048, "vocab": 131072, "top": 5, "type": "bf16",
         "temperature": 1.0},
        # learning from rewards, with a term for the entropy; rows that start at odd addresses
        {"name": "score_train", "kind": "score_train", "rows": 1037, "vocab": 50021, "top": 0, "type": "f16",
         "temperature": 0.7},
        # the parameters of one small readout
        {"name": "adamw_small", "kind": "adamw", "tensors": 14, "elements": 200000, "bits": 32, "type": "f32",
         "grad": "f32"},
        # a large model's, its states in 8 bits
        {"name": "adamw_large", "kind": "adamw", "tensors": 300, "elements": 150000000, "bits": 8, "type": "bf16",
         "grad": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["recur", "recur_train", "recur_step", "norm", "norm_train", "norm_train", "score", "score_train",
                       "adamw", "adamw"])
    case = {"kind": kind, "type": rng.choice(["f32", "bf16", "f16"])}
    if kind == "recur_step":
        case |= {"batch": _log(rng, 1, 512), "channels": _log(rng, 1, 8192)}
        case["slots"] = case["batch"] + rng.randint(0, 30)
    elif kind in ("recur", "recur_train"):
        case |= {"batch": _log(rng, 1, 64), "time": _log(rng, 1, 65536), "channels": _log(rng, 1, 8192)}
        while case["time"] > 1 and case["batch"] * case["time"] * case["channels"] > 1 << 25:
            case["time"] //= 2
        case |= {"ragged": rng.random() < 0.5, "state": rng.random() < 0.5}
    elif kind in ("norm", "norm_train"):
        case |= {"rows": _log(rng, 1, 65536), "width": _log(rng, 4, 40000)}
        while case["rows"] > 1 and case["rows"] * case["width"] > 1 << 26:
            case["rows"] //= 2
    elif kind in ("score", "score_train"):
        case |= {"rows": _log(rng, 1, 4096), "vocab": _log(rng, 2, 262144)}
        while case["rows"] > 1 and case["rows"] * case["vocab"] > 1 << 26:
            case["rows"] //= 2
        case |= {"top": min(case["vocab"], rng.choice([0, 1, 5, 20, rng.randint(1, 128)])),
                 "temperature": rng.choice([0.5, 1.0, 1.0, 2.0])}
    else:
        case |= {"tensors": _log(rng, 1, 300), "bits": rng.choice([8, 32]), "grad": rng.choice(["f32", case["type"]])}
        case["elements"] = max(case["tensors"], _log(rng, 1, 50000000))
    return case


def _sizes(case):
    """Elements of each tensor: a few large ones hold most of them, many are vectors."""
    rng = random.Random(case["tensors"] * 1000003 + case["elements"])
    part = [math.exp(rng.uniform(0.0, 8.0)) for _ in range(case["tensors"])]
    whole = sum(part)
    return [max(1, int(case["elements"] * p / whole)) for p in part]


# ------------------------------------------------------------------------------ inputs
def _normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    kind = case["kind"].split("_")[0]
    make = {"recur": _prepare_recur, "norm": _prepare_norm, "score": _prepare_score, "adamw": _prepare_adamw}
    return {"case": case} | make[kind](case, gen)


def _prepare_recur(case, gen):
    b, c, dtype = case["batch"], case["channels"], TYPES[case["type"]]
    # channels remember for 4 steps to 1024; values and gates come out of one projection, side by side
    keep = torch.log(4.0 * 256.0 ** (torch.arange(c, device=DEV) / max(c - 1, 1)) - 1.0)
    one = torch.randn(b, case.get("time", 1), 2, c, generator=gen, device=DEV)
    one[:, :, 1] = keep + 0.5 * one[:, :, 1]
    one = one.to(dtype).flatten(2)
    s = {"x": one[..., :c], "gate": one[..., c:], "state": None, "lengths": None}
    if case["kind"] == "recur_step":
        s["x"], s["gate"] = s["x"][:, 0], s["gate"][:, 0]
        # the pool has a row more than its slots, which the plain form gives to what has no slot
        s["pool"] = _normal(gen, case["slots"] + 1, c)
        s["state"] = s["pool"][:-1]
        slots = torch.randperm(case["slots"], generator=gen, device=DEV)[:b]
        # a sequence that has ended keeps its place in the batch, without a slot
        if b > 4:
            slots = torch.where(torch.rand(b, generator=gen, device=DEV) < 0.05, -1, slots)
        s["slots"] = slots.to(torch.int32)
        return s
    if case["state"]:
        s["state"] = _normal(gen, b, c)
    if case["ragged"]:
        lengths = torch.randint(0, case["time"] + 1, (b,), generator=gen, device=DEV)
        lengths[0] = case["time"]
        if b > 2:
            lengths[1], lengths[2] = 0, 1
        s["lengths"] = lengths.to(torch.int32)
    if case["kind"] == "recur_train":
        s["do"] = _normal(gen, b, case["time"], c, dtype=dtype)
        s["dstate"] = _normal(gen, b, c) if case["state"] else None
    return s


def _prepare_norm(case, gen):
    rows, width, dtype = case["rows"], case["width"], TYPES[case["type"]]
    x = _normal(gen, rows, width)
    if case["type"] == "f32":
        x = x * 8.0 - 65.0                  # voltages
    else:
        # activations: rows of different sizes, some channels larger than the others
        x = x * torch.exp(0.5 * _normal(gen, rows, 1)) * torch.exp(0.7 * _normal(gen, width)) + 0.3 * _normal(gen, width)
    s = {"x": x.to(dtype), "weight": 1.0 + 0.2 * _normal(gen, width), "bias": 0.2 * _normal(gen, width)}
    if case["kind"] == "norm_train":
        s["dy"] = _normal(gen, rows, width, dtype=dtype)
    return s


def _prepare_score(case, gen):
    rows, vocab, dtype = case["rows"], case["vocab"], TYPES[case["type"]]
    # a trained model's logits: most of the mass on a small part of the vocabulary
    logits = _normal(gen, rows, vocab, scale=3.0)
    # answers drawn from what the model gave
    token = (logits - torch.log(-torch.log(torch.rand(rows, vocab, generator=gen, device=DEV).clamp(1e-7, 1 - 1e-7)))).argmax(1)
    # some rows may only answer from a part of the vocabulary
    some = torch.rand(rows, 1, generator=gen, device=DEV) < (0.1 if vocab >= 1024 else 0.0)
    shut = some & (torch.rand(vocab, generator=gen, device=DEV) < 0.7)
    shut.scatter_(1, token[:, None], False)
    logits = torch.where(shut, -torch.inf, logits)
    # padding has no token
    token = torch.where(torch.rand(rows, generator=gen, device=DEV) < 0.02, -1, token)
    s = {"logits": logits.to(dtype), "tokens": token}
    if case["kind"] == "score_train":
        # advantages, averaged over the rows; in f16 scaled up so that gradients keep their bits
        size = (1024.0 if case["type"] == "f16" else 1.0) / rows
        s["dlogprob"] = _normal(gen, rows, scale=size)
        s["dentropy"] = torch.full((rows,), 0.01 * size, device=DEV)
    return s


def _prepare_adamw(case, gen):
    sizes, dtype, grad = _sizes(case), TYPES[case["type"]], TYPES[case["grad"]]
    # parameters lie one after another in one buffer, each from a multiple of BLOCK; so do their moments
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + -(-n // BLOCK) * BLOCK)
    whole = starts.pop()
    flat = torch.zeros(whole, dtype=dtype, device=DEV)
    s = {"flat": flat, "params": [flat[at:at + n] for at, n in zip(starts, sizes)], "grads": [], "starts": starts,
         "m": torch.zeros(whole, dtype=torch.float8_e4m3fn if case["bits"] == 8 else torch.float32, device=DEV),
         "m_scale": torch.zeros(whole // BLOCK, device=DEV) if case["bits"] == 8 else None,
         # matrices decay, vectors do not
         "decay": [0.01 if n > 4096 else 0.0 for n in sizes],
         "step": torch.full((1,), 99, dtype=torch.int64, device=DEV),
         # what clipping the gradients' norm gave
         "clip": torch.rand(1, generator=gen, device=DEV) * 0.5 + 0.5}
    s |= {"v": torch.zeros_like(s["m"]), "v_scale": None if s["m_scale"] is None else torch.zeros_like(s["m_scale"])}
    for i, n in enumerate(sizes):
        size = torch.exp(_normal(gen, n)) * 1e-3            # an element's usual gradient
        s["params"][i].copy_(_normal(gen, n, scale=0.05))
        s["grads"].append((size * _normal(gen, n)).to(grad))
        _put_moments(s, i, 0.3 * size * _normal(gen, n), (size * torch.exp(0.2 * _normal(gen, n))) ** 2)
    if own:
        from heliox_amd import readout

        s["handle"] = readout.adamw_state(s["params"], bits=case["bits"])
        for name in ("step", "m", "v", "m_scale", "v_scale"):
            here = s.pop(name)
            if here is not None:
                getattr(s["handle"], name).copy_(here)
    return s


def _put_moments(s, i, m, v):
    """Tensor i's moments, to where they are held."""
    at, n = s["starts"][i], s["params"][i].numel()
    if s["m_scale"] is not None:
        for name, x, floor in (("m", m, False), ("v", v.sqrt(), True)):
            code, scale = _to8(x, floor)
            s[name][at:at + n].copy_(code)
            s[name + "_scale"][at // BLOCK:at // BLOCK + scale.numel()].copy_(scale)
    else:
        s["m"][at:at + n].copy_(m)
        s["v"][at:at + n].copy_(v)


def _moments(s, i):
    """Tensor i's moments as they are held: m, and v (in 8 bits: its root)."""
    at, n = s["starts"][i], s["params"][i].numel()
    if s["m_scale"] is None:
        return s["m"][at:at + n], s["v"][at:at + n]
    scale = [s[name][at // BLOCK:at // BLOCK + -(-n // BLOCK)].repeat_interleave(BLOCK)[:n] for name in ("m_scale", "v_scale")]
    return s["m"][at:at + n].float() * scale[0], s["v"][at:at + n].float() * scale[1]


def _to8(x, floor=False):
    """Blocks of BLOCK elements in 8 bits relative to the largest of them, and their scales; with
    floor, what is not zero is at least the smallest value."""
    n = x.numel()
    x = torch.nn.functional.pad(x, (0, -n % BLOCK)).view(-1, BLOCK)
    top = x.abs().amax(1, keepdim=True)
    live = top >= 2.0 ** -100
    r = torch.where(live, x / torch.where(live, top, 1.0) * TOP8, 0.0)
    if floor:
        r = torch.where(r > 0, r.clamp(min=LEAST8), r)
    scale = torch.where(live, top / TOP8, 0.0)[:, 0]
    return r.float().to(torch.float8_e4m3fn).flatten()[:n], scale.float()


# --------------------------------------------------------------------------------- run
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from heliox_amd import readout

    case, kind = s["case"], s["case"]["kind"]
    if kind == "recur_step":
        return {"o": readout.gated_recurrence_step(s["x"], s["gate"], s["state"], slots=s["slots"]), "state": s["state"]}
    if kind in ("recur", "recur_train"):
        how = {"initial_state": s["state"], "lengths": s["lengths"]}
        o, end = readout.gated_recurrence(s["x"], s["gate"], **how)
        got = {"o": o, "end": end}
        if kind == "recur_train":
            got["dx"], got["dgate"], d0 = readout.gated_recurrence_grad(s["x"], s["gate"], s["do"], dstate=s["dstate"],
                                                                        **how)
            if d0 is not None:
                got["dinitial"] = d0
        return got
    if kind in ("norm", "norm_train"):
        y, mean, rstd = readout.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
        if kind == "norm":
            return {"y": y}
        dx, dw, db = readout.layer_norm_grad(s["x"], s["weight"], mean, rstd, s["dy"])
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    if kind in ("score", "score_train"):
        tau = case["temperature"]
        got = readout.token_logprobs(s["logits"], s["tokens"], temperature=tau, top=case["top"])
        out = {"logprob": got.logprob, "entropy": got.entropy, "top_logprob": got.top_logprob, "top_index": got.top_index}
        if kind == "score_train":
            out["grad"] = readout.token_logprobs_grad(s["logits"], s["tokens"], got, s["dlogprob"], s["dentropy"],
                                                      temperature=tau)
        return out
    readout.adamw_step(s["params"], s["grads"], s["handle"], lr=LR, betas=BETAS, eps=ADAM_EPS, weight_decay=s["decay"],
                       grad_scale=s["clip"])
    held = s["handle"]
    return _adamw_out(s["flat"], held.m, held.v, held.m_scale, held.v_scale, held.step)


def _adamw_out(flat, m, v, m_scale, v_scale, step):
    out = {"params": flat, "m": m, "v": v, "step": step}
    return out if m_scale is None else out | {"m_scale": m_scale, "v_scale": v_scale}


def _run_plain(s):
    plain = {"recur_step": _plain_step, "recur": _plain_recur, "recur_train": _plain_recur, "norm": _plain_norm,
             "norm_train": _plain_norm, "score": _plain_score, "score_train": _plain_score, "adamw": _plain_adamw}
    return plain[s["case"]["kind"]](s)


def _plain_step(s):
    pool, kind = s["pool"], s["x"].dtype
    live = s["slots"] >= 0
    at = torch.where(live, s["slots"], s["case"]["slots"]).long()
    x, u = s["x"].float(), s["gate"].float()
    h = torch.sigmoid(u) * pool[at] + torch.sigmoid(-u) * x
    pool[at] = h
    return {"o": torch.where(live[:, None], h, 0.0).to(kind), "state": s["state"]}


def _doubling(a, b):
    """y_t = a_t y_{t-1} + b_t over dimension 1 from y = 0, and the running products of a."""
    d = 1
    while d < a.shape[1]:
        b = torch.cat([b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return a, b


def _scan(a, b, first):
    """y_t = a_t y_{t-1} + b_t, y_{-1} = first, for (B, T, C) arrays: chunks of CHUNK steps by
    themselves, then what enters each."""
    batch, t, c = a.shape
    n = -(-t // CHUNK)
    pad = (0, 0, 0, n * CHUNK - t)
    a = torch.nn.functional.pad(a, pad, value=1.0).reshape(batch * n, CHUNK, c)
    b = torch.nn.functional.pad(b, pad).reshape(batch * n, CHUNK, c)
    a, b = _doubling(a, b)
    ends_a, ends_b = _doubling(a[:, -1].view(batch, n, c), b[:, -1].view(batch, n, c))
    ends = ends_a * first[:, None] + ends_b
    enter = torch.cat([first[:, None], ends[:, :-1]], 1).reshape(batch * n, 1, c)
    return (a * enter + b).view(batch, n * CHUNK, c)[:, :t]


def _plain_recur(s):
    x, u, kind = s["x"].float(), s["gate"].float(), s["x"].dtype
    batch, t, c = x.shape
    first = s["state"] if s["state"] is not None else torch.zeros(batch, c, device=x.device)
    lengths = s["lengths"].long() if s["lengths"] is not None else torch.full((batch,), t, device=x.device)
    live = (torch.arange(t, device=x.device) < lengths[:, None])[..., None]
    a, z = torch.sigmoid(u), torch.sigmoid(-u)
    # past its length a sequence stands still
    h = _scan(torch.where(live, a, 1.0), torch.where(live, z * x, 0.0), first)
    got = {"o": torch.where(live, h, 0.0).to(kind), "end": h[:, -1].contiguous()}
    if s["case"]["kind"] == "recur":
        return got
    before = torch.cat([first[:, None], h[:, :-1]], 1)
    last = s["dstate"] if s["dstate"] is not None else torch.zeros_like(first)
    keep = torch.where(live, a, 1.0)
    later = torch.cat([keep[:, 1:], torch.ones_like(keep[:, :1])], 1)
    back = _scan(later.flip(1), torch.where(live, s["do"].float(), 0.0).flip(1), last).flip(1)
    got["dx"] = torch.where(live, z * back, 0.0).to(kind)
    got["dgate"] = torch.where(live, a * z * back * (before - x), 0.0).to(kind)
    return got | {"dinitial": keep[:, 0] * back[:, 0]} if s["state"] is not None else got


def _plain_norm(s):
    x, w, kind = s["x"].float(), s["weight"], s["x"].dtype
    off = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((off * off).mean(1, keepdim=True) + EPS)
    xhat = off * rstd
    y = (xhat * w + s["bias"]).to(kind)
    if s["case"]["kind"] == "norm":
        return {"y": y}
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(kind), "dweight": (dy * xhat).sum(0), "dbias": dy.sum(0)}


def _plain_score(s):
    tau, k, kind = s["case"]["temperature"], s["case"]["top"], s["logits"].dtype
    x = s["logits"].float()
    z = (x - x.amax(1, keepdim=True)) / tau
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    q, logq = e / total, z - total.log()
    entropy = -torch.where(q > 0, q * logq, 0.0).sum(1)
    here = s["tokens"] >= 0
    at = s["tokens"].clamp(min=0)[:, None]
    # the largest first, the lowest index where they are equal: one whole number for both
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * 2 ** 32 - torch.arange(x.shape[1], device=x.device)
    top = torch.topk(key, k, dim=1).values
    index = -top % 2 ** 32
    got = {"logprob": torch.where(here, logq.gather(1, at)[:, 0], 0.0), "entropy": entropy,
           "top_logprob": logq.gather(1, index), "top_index": index}
    if s["case"]["kind"] == "score":
        return got
    pull = torch.where(here, s["dlogprob"], 0.0)[:, None]
    turn = s["dentropy"][:, None]
    grad = -q * (pull + turn * (torch.where(q > 0, logq, 0.0) + entropy[:, None]))
    grad = grad.scatter_add_(1, at, pull) / tau
    return got | {"grad": grad.to(kind)}


def _plain_adamw(s):
    eight, (b1, b2) = s["case"]["bits"] == 8, BETAS
    s["step"] += 1
    t = s["step"].double()
    c1, c2 = (1 - b1 ** t).float(), (1 - b2 ** t).float()
    for i, (p, g, decay) in enumerate(zip(s["params"], s["grads"], s["decay"])):
        g = g.float() * s["clip"]
        m, v = _moments(s, i)
        m = b1 * m + (1 - b1) * g
        v = b2 * (v * v if eight else v) + (1 - b2) * g * g
        p.copy_(p.float() * (1 - LR * decay) - LR * (m / c1) / ((v / c2).sqrt() + ADAM_EPS))
        _put_moments(s, i, m, v)
    return _adamw_out(s["flat"], s["m"], s["v"], s["m_scale"], s["v_scale"], s["step"])


# -------------------------------------------------------------------------------- work
def work(case):
    kind, size = case["kind"], TYPES[case["type"]].itemsize
    if kind == "adamw":
        n = sum(_sizes(case))
        states = 16 * n if case["bits"] == 32 else 4 * n + 16 * sum(-(-m // BLOCK) for m in _sizes(case))
        return {"bytes": n * (2 * size + TYPES[case["grad"]].itemsize) + states, "flops": 16 * n}
    if kind == "recur_step":
        n = case["batch"] * case["channels"]
        return {"bytes": n * (3 * size + 8), "flops": 4 * n}
    if kind in ("recur", "recur_train"):
        n, states = case["batch"] * case["time"] * case["channels"], 4 * case["batch"] * case["channels"]
        if kind == "recur":
            return {"bytes": 3 * n * size + states * (2 if case["state"] else 1), "flops": 4 * n}
        return {"bytes": 6 * n * size + states * (4 if case["state"] else 1), "flops": 14 * n}
    n = case["rows"] * case.get("width", case.get("vocab", 0))
    if kind == "norm":
        return {"bytes": 2 * n * size + 8 * case["width"], "flops": 8 * n}
    if kind == "norm_train":
        return {"bytes": 4 * n * size + 16 * case["width"] + 16 * case["rows"], "flops": 24 * n}
    if kind == "score":
        return {"bytes": n * size + case["rows"] * (16 + 12 * case["top"]), "flops": 6 * n}
    return {"bytes": 2 * n * size + case["rows"] * (24 + 12 * case["top"]), "flops": 12 * n}


# ------------------------------------------------------------------------------- exact
def exact(case, seed):
    global own
    was, own = own, False                   # inputs alone, without a handle
    try:
        s = prepare(case, seed)
    finally:
        own = was
    kind = case["kind"].split("_")[0]
    return {"recur": _exact_recur, "norm": _exact_norm, "score": _exact_score, "adamw": _exact_adamw}[kind](s)


def _exact_recur(s):
    """The recurrence itself, one step after another."""
    x, u = s["x"].double(), s["gate"].double()
    a = 1 / (1 + torch.exp(-u))
    if s["case"]["kind"] == "recur_step":
        state, o = s["state"].double(), torch.zeros_like(x)
        for i, at in enumerate(s["slots"].tolist()):
            if at >= 0:
                state[at] = o[i] = a[i] * state[at] + (1 - a[i]) * x[i]
        return {"o": o, "state": state}
    batch, steps, c = x.shape
    first = s["state"].double() if s["state"] is not None else torch.zeros(batch, c, dtype=torch.float64, device=x.device)
    ends = s["lengths"].tolist() if s["lengths"] is not None else [steps] * batch
    order = sorted(range(batch), key=lambda i: -ends[i])            # the longest first: those alive are a prefix
    alive = [sum(e > t for e in ends) for t in range(steps)]
    x, a, h = x[order], a[order], first[order].clone()
    o, before = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(steps):
        n = alive[t]
        before[:n, t] = h[:n]
        h[:n] += (1 - a[:n, t]) * (x[:n, t] - h[:n])
        o[:n, t] = h[:n]
    back = [order.index(i) for i in range(batch)]
    got = {"o": o[back], "end": h[back]}
    if s["case"]["kind"] == "recur":
        return got
    l = s["dstate"].double()[order] if s["dstate"] is not None else torch.zeros_like(h)
    do, dx, du = s["do"].double()[order], torch.zeros_like(x), torch.zeros_like(x)
    for t in reversed(range(steps)):
        n = alive[t]
        l[:n] += do[:n, t]
        dx[:n, t] = (1 - a[:n, t]) * l[:n]
        du[:n, t] = l[:n] * (before[:n, t] - x[:n, t]) * a[:n, t] * (1 - a[:n, t])
        l[:n] *= a[:n, t]
    got |= {"dx": dx[back], "dgate": du[back]}
    return got | {"dinitial": l[back]} if s["state"] is not None else got


def _exact_norm(s):
    train, rows = s["case"]["kind"] == "norm_train", s["x"].shape[0]
    w, b = s["weight"].double(), s["bias"].double()
    got = {"y": []} | ({"dx": []} if train else {})
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    for lo in range(0, rows, 4096):
        x = s["x"][lo:lo + 4096].double()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        sd = torch.sqrt(var + EPS)
        n = (x - mean) / sd
        got["y"].append(n * w + b)
        if train:
            dy = s["dy"][lo:lo + 4096].double()
            dw += torch.einsum("rw,rw->w", dy, n)
            db += dy.sum(0)
            c = dy * w / sd
            got["dx"].append(c - c.mean(1, keepdim=True) - n * torch.einsum("rw,rw->r", c, n)[:, None] / x.shape[1])
    got = {k: torch.cat(v) for k, v in got.items()}
    return got | {"dweight": dw, "dbias": db} if train else got


def _exact_score(s):
    tau, k, n = s["case"]["temperature"], s["case"]["top"], s["logits"].shape[0]
    train = s["case"]["kind"] == "score_train"
    parts = {"logprob": [], "entropy": [], "top_logprob": []} | ({"grad": []} if train else {})
    for lo in range(0, n, 256):
        logq = torch.log_softmax(s["logits"][lo:lo + 256].double() / tau, dim=1)
        q = logq.exp()
        token = s["tokens"][lo:lo + 256]
        row = torch.arange(len(token), device=token.device)
        there = (token >= 0).double()
        gain = torch.where(q > 0, logq, 0.0)
        h = -(q * gain).sum(1)
        parts["logprob"].append(torch.where(token >= 0, logq[row, token], 0.0))
        parts["entropy"].append(h)
        parts["top_logprob"].append(torch.sort(logq, dim=1, descending=True).values[:, :k])
        if train:
            lp, e = s["dlogprob"][lo:lo + 256].double() * there, s["dentropy"][lo:lo + 256].double()
            g = -q * (lp[:, None] + e[:, None] * (gain + h[:, None]))
            g[row, token] += lp
            parts["grad"].append(g / tau)
    return {name: torch.cat(v) for name, v in parts.items()} | {"top_index": None}


def _exact8(x, floor=False):
    """The nearest numbers with four bits after the first, even where two are as near, from 2^-9 to 448."""
    n = x.numel()
    y = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    y[:n] = x
    y = y.view(-1, BLOCK)
    scale = y.abs().max(1).values / 448
    y = torch.where(scale[:, None] > 0, y / scale[:, None].clamp(min=1e-300), 0.0)
    unit = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))).clamp(max=8) - 3)
    z = torch.round(y / unit) * unit
    if floor:
        z = torch.where((y > 0) & (z < 2.0 ** -9), 2.0 ** -9, z)
    return z.flatten()[:n], scale


def _exact_adamw(s):
    eight, (b1, b2) = s["case"]["bits"] == 8, BETAS
    t = int(s["step"]) + 1
    clip = s["clip"].double()
    out = {name: torch.zeros(s["m"].shape, dtype=torch.float64, device=clip.device) for name in ("params", "m", "v")}
    if eight:
        out |= {name: torch.zeros_like(s[name], dtype=torch.float64) for name in ("m_scale", "v_scale")}
    for p, g, at, decay in zip(s["params"], s["grads"], s["starts"], s["decay"]):
        here = slice(at, at + p.numel())
        m, v, g = s["m"][here].double(), s["v"][here].double(), g.double() * clip
        if eight:
            of = torch.arange(at, at + p.numel(), device=p.device) // BLOCK
            m, v = m * s["m_scale"].double()[of], (v * s["v_scale"].double()[of]) ** 2
        m, v = m + (1 - b1) * (g - m), v + (1 - b2) * (g * g - v)
        step = m / (1 - b1 ** t) / (torch.sqrt(v / (1 - b2 ** t)) + ADAM_EPS)
        out["params"][here] = p.double() - LR * (step + decay * p.double())
        if eight:
            (m, ms), (v, vs) = _exact8(m), _exact8(v.sqrt(), floor=True)
            blocks = slice(at // BLOCK, at // BLOCK + ms.numel())
            out["m_scale"][blocks], out["v_scale"][blocks] = ms, vs
        out["m"][here], out["v"][here] = m, v
    return out | {"step": None}
