"""References in 64 bits for the readout operators, step by step and row by row."""
import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attention(q, k, v, log_decay, scale, initial=None, lengths=None, do=None, dend=None):
    """The recurrence; with do its gradients too.  Inputs of any type and device; float64 on the CPU out."""
    heads, kind = log_decay.shape[0], torch.float64
    wide = lambda x: x.detach().cpu().to(kind).repeat_interleave(heads // x.shape[2], dim=2)  # noqa: E731
    nq, nk, nv = q.shape[2], k.shape[2], v.shape[2]
    q, k, v = wide(q), wide(k), wide(v)
    batch, steps, _, dk = q.shape
    dv = v.shape[-1]
    gamma = log_decay.detach().cpu().to(kind).exp()[:, None, None]
    o = torch.zeros(batch, steps, heads, dv, dtype=kind)
    dq, dk_, dv_ = (torch.zeros(batch, steps, heads, n, dtype=kind) for n in (dk, dk, dv))
    end = torch.zeros(batch, heads, dk, dv, dtype=kind) if initial is None else initial.cpu().to(kind).clone()
    dinitial = torch.zeros_like(end)
    for i in range(batch):
        n = steps if lengths is None else int(lengths[i])
        s = end[i].clone()
        for t in range(n):
            s = gamma * s + k[i, t, :, :, None] * v[i, t, :, None, :]
            o[i, t] = scale * torch.einsum("hk,hkv->hv", q[i, t], s)
            if do is not None:
                dq[i, t] = scale * torch.einsum("hv,hkv->hk", do[i, t].cpu().to(kind), s)
        end[i] = s
        if do is None:
            continue
        g = torch.zeros_like(s) if dend is None else dend[i].cpu().to(kind)
        for t in reversed(range(n)):
            g = g + scale * q[i, t, :, :, None] * do[i, t].cpu().to(kind)[:, None, :]
            dk_[i, t] = torch.einsum("hkv,hv->hk", g, v[i, t])
            dv_[i, t] = torch.einsum("hkv,hk->hv", g, k[i, t])
            g = gamma * g
        dinitial[i] = g
    if do is None:
        return o, end
    share = lambda x, n: x.unflatten(2, (n, -1)).sum(3)  # noqa: E731
    return o, end, share(dq, nq), share(dk_, nk), share(dv_, nv), dinitial


def distill(logits, index, teacher, tau, lse=None, weight=None):
    """Loss and gradient, row by row, float64 on the CPU."""
    kind = torch.float64
    x, t = logits.detach().cpu().to(kind) / tau, teacher.detach().cpu().to(kind) / tau
    rows, vocab = x.shape
    loss, grad = torch.zeros(rows, dtype=kind), torch.zeros(rows, vocab, dtype=kind)
    for i in range(rows):
        entries = [(int(j), t[i, n]) for n, j in enumerate(index[i].tolist()) if 0 <= j < vocab]
        if not entries:
            continue
        logq = x[i] - torch.logsumexp(x[i], 0)
        z = torch.stack([e for _, e in entries])
        norm = torch.logsumexp(z, 0) if lse is None else lse[i].cpu().to(kind)
        p = torch.zeros(vocab, dtype=kind)
        for (j, e) in entries:
            share = torch.exp(e - norm) if e > -torch.inf else torch.zeros((), dtype=kind)
            p[j] += share
            if share > 0:
                loss[i] += share * (e - norm - logq[j])
        members = sorted({j for j, _ in entries})
        outside = torch.ones(vocab, dtype=torch.bool)
        outside[members] = False
        total = p.sum()
        q = logq.exp()
        factor = torch.full((vocab,), float(total), dtype=kind)
        if lse is not None:
            pr, qr = 1 - total, q[outside].sum()
            if pr > 0 and qr > 0:
                loss[i] += pr * torch.log(pr / qr)
                factor += pr
                factor[outside] -= pr / qr
        grad[i] = q * factor - p
    w = torch.ones(rows, dtype=kind) if weight is None else weight.cpu().to(kind)
    return loss * tau * tau, grad * tau * w[:, None]


def masses(row, temperature, top_k, top_p, min_p):
    """A row's masses in 64 bits, and which places stay; (mass, stays, slack): `slack` is the share by which
    a bound on sums may be missed because the library's weights are fp32."""
    x = row.detach().cpu().double()
    x = torch.where(x.isnan(), -torch.inf, x)
    if temperature <= 0:
        top_k, temperature = 1, 1.0
    e = torch.exp((x - x.max()) / temperature)
    m = torch.floor(e * 2.0 ** 40)
    order = torch.sort(x, descending=True, stable=True).indices
    n = top_k if 0 < top_k < x.numel() else x.numel()
    if top_p < 1:
        run = m[order[:n]].cumsum(0)
        n = max(1, 1 + int((run[:-1] < top_p * run[-1]).sum()))
    stays = torch.zeros(x.numel(), dtype=torch.bool)
    stays[order[:n]] = True
    return m, stays & (e >= min(min_p, 1.0))


def rel(got, want):
    """2-norm of the difference over that of the result."""
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert bool(torch.isfinite(got).all())
    norm = float(want.norm())
    off = float((got - want).norm())
    return off / norm if norm else off


def captured(call, change):
    """The call, captured once and replayed three times with other inputs and its own eager runs in
    between, gives what it gives by itself."""
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for n in range(3):
        change(torch.Generator().manual_seed(n))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [x.clone() for x in got]
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, want)), n
