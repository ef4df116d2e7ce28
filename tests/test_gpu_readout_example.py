"""The readout operators together, as examples/teach_readout.py runs them on a network: the
gradient by the voltages against differences, a falling loss, and the closed loop against the
whole recording."""
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
    spec = importlib.util.spec_from_file_location("teach_readout", os.path.join(ROOT, "examples", "teach_readout.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_gradient_by_the_voltages(example):
    """Central differences along a random way.  The loss of 60 ticks is smooth on the scale of a
    step of 0.02 mV (1e-3 of the readout's range): the differences' own error is under 1e-4 of
    the gradient's size along the way, the loss's fp32 rounding 2^-20 of it over the step."""
    ticks, cells, classes = 60, 3, 40
    gen = torch.Generator().manual_seed(0)
    v = (torch.randn(ticks, cells, generator=gen) * 8 - 60).cuda()
    student = example.Readout(cells, classes, seed=2)
    full = torch.randn(ticks, classes, generator=gen).cuda()
    best, at = torch.topk(full, 6, dim=1)
    lse = torch.logsumexp(full, 1)

    def loss(v):
        return float(readout.distill_loss(student.forward(v), at, best, teacher_lse=lse).double().sum())

    logits = student.forward(v)
    _, dlogits = readout.distill_loss_grad(logits, at, best, teacher_lse=lse)
    dv = student.backward(dlogits)[2]
    way = torch.randn(ticks, cells, generator=gen).cuda()
    step = 0.02
    diff = (loss(v + step * way) - loss(v - step * way)) / (2 * step)
    exact = float((dv.double() * way.double()).sum())
    size = float(dv.double().norm() * way.double().norm())
    assert abs(diff - exact) <= 1e-4 * size + 2.0 ** -20 * loss(v) / step


def test_the_network_learns_from_its_teacher(example):
    lines = []
    network, student, losses = example.teach(cells=3, ticks=60, passes=6, say=lines.append)
    assert len(lines) == 6 and np.all(np.isfinite(losses))
    assert losses[-1] < 0.9 * losses[0]


def test_closed_loop_gives_the_recordings_logits(example):
    """Tick by tick the readout gives what it gives for the recording of the same run: both read
    the same voltages, in fp32, the sums of 20 ticks in another order."""
    network = example.Network(3, 20)
    student = example.Readout(3, 50, seed=3)
    whole = student.forward(network.run())
    tokens, logits = example.answer(network, student, ticks=20)
    assert tokens.shape == (20,) and bool(((tokens >= 0) & (tokens < 50)).all())
    scale = float(whole.abs().max())
    assert float((logits - whole).abs().max()) <= 1e-5 * scale
