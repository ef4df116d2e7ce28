"""Layer norm, the gated recurrence, log probabilities and AdamW together, as
examples/recurrent_readout.py runs them on a network: gradients against differences, a training
run, and the closed loop against the whole recording."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from heliox_amd import readout

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("recurrent_readout", os.path.join(ROOT, "examples", "recurrent_readout.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def in_64_bits(student, voltages, token, earned, entropy_weight, parameters):
    """The example's loss from its definitions, in torch and 64 bits, which makes its gradients."""
    w, b, w_in, w_out = parameters
    off = voltages - voltages.mean(1, keepdim=True)
    n = off / torch.sqrt((off ** 2).mean(1, keepdim=True) + 1e-5) * w + b
    value, gate = (n @ w_in).split(student.channels, dim=-1)
    a = torch.sigmoid(gate + student.keep.cpu().double())
    h, o = torch.zeros(student.channels, dtype=torch.float64), []
    for t in range(len(token)):
        h = a[t] * h + (1 - a[t]) * value[t]
        o.append(h)
    logq = torch.log_softmax(torch.stack(o) @ w_out, 1)
    gain = earned[torch.arange(len(token)), token]
    gain = gain - gain.mean()
    return -(gain * logq[torch.arange(len(token)), token] - entropy_weight * (logq.exp() * logq).sum(1)).mean()


def test_gradients(example):
    """Of every parameter and of the voltages, through all of the operators.  fp32 throughout: each
    result is off by some dozens of roundings, 2^-18 of a gradient's norm."""
    ticks, cells, classes = 70, 5, 12
    gen = torch.Generator().manual_seed(0)
    v = (torch.randn(ticks, cells, generator=gen) * 8 - 60).cuda()
    student = example.Readout(cells, classes, channels=20, seed=2)
    earned = example.reward_of(ticks, classes)
    token = torch.randint(classes, (ticks,), generator=gen).cuda()
    dlogits, _, _ = example.gradient(student.forward(v), token, earned, 0.05)
    grads, dv = student.backward(dlogits)
    wide = [p.detach().cpu().double().requires_grad_() for p in student.parameters()]
    voltages = v.cpu().double().requires_grad_()
    in_64_bits(student, voltages, token.cpu(), earned.cpu().double(), 0.05, wide).backward()
    for got, want in zip([*grads, dv], [p.grad for p in wide] + [voltages.grad]):
        assert float((got.cpu().double() - want).norm()) <= 2.0 ** -15 * float(want.norm())


def test_it_trains(example):
    lines = []
    network, student, history = example.train(cells=3, ticks=60, passes=4, say=lines.append)
    assert len(lines) == 4 and np.all(np.isfinite(history))
    assert int(student.state.step) == 4 and all(bool(torch.isfinite(p).all()) for p in student.parameters())


def test_closed_loop_gives_the_recordings_logits(example):
    """Tick by tick the readout gives what it gives for the recording of the same run, and what its
    answers' logarithms say is what the recording's say."""
    network = example.Network(3, 20)
    student = example.Readout(3, 30, seed=3)
    whole = student.forward(network.run())
    tokens, scored, logits = example.answer(network, student, ticks=20)
    scale = float(whole.abs().max())
    assert float((logits - whole).abs().max()) <= 1e-5 * scale
    at_once = readout.token_logprobs(logits, tokens, top=3)
    # A row's 30 weights are added in an order that its address in 16 bytes decides: each of 30 sums is off by
    # at most 2^-24 of the whole, each weight by 4 times that, so a logarithm by 34 x 2^-24 and its own
    # rounding, and two of them are apart by twice that; an entropy adds as many terms of up to log 30 = 3.4.
    for t, one in enumerate(scored):
        assert torch.equal(one.top_index[0], at_once.top_index[t])
        for name, size in (("logprob", 1.0), ("top_logprob", 1.0), ("entropy", 1.0 + 2 * 3.4)):
            a, b = getattr(one, name)[0], getattr(at_once, name)[t]
            assert float((a - b).abs().max()) <= 2 * 2.0 ** -24 * (34 * size + float(b.abs().max()))
