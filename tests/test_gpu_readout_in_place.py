"""Tensors that a call writes in place: a backward pass that kept their old values says so instead of going on with others."""
import pytest
import torch

from heliox_amd import readout

pytestmark = pytest.mark.gpu


def recurrence_step(state):
    x = torch.ones(2, 3, device="cuda")
    readout.gated_recurrence_step(x, x, state)


def attention_step(state):
    x = torch.ones(2, 1, 3, device="cuda")
    readout.linear_attention_step(x, x, x[..., :1], torch.zeros(1, device="cuda"), state.view(2, 1, 3, 1))


def logprobs_grad(logits):
    tokens = torch.zeros(2, dtype=torch.int64, device="cuda")
    readout.token_logprobs_grad(logits, tokens, readout.token_logprobs(logits, tokens), torch.ones(2, device="cuda"), out=logits)


def distill_grad(logits):
    teacher = torch.zeros(2, 1, dtype=torch.int64, device="cuda"), torch.ones(2, 1, device="cuda")
    readout.distill_loss_grad(logits, *teacher, out=logits)


def optimizer(p):
    readout.adamw_step([p], [torch.ones(2, 3, device="cuda")], readout.adamw_state([p]), lr=0.1)


CALLS = [recurrence_step, attention_step, logprobs_grad, distill_grad, optimizer]


@pytest.mark.parametrize("call", CALLS)
def test_a_graph_of_the_old_values_is_refused(call):
    at = torch.zeros(2, 3, device="cuda")
    w = torch.ones(2, 3, device="cuda", requires_grad=True)
    y = (at * w).sum()                                          # keeps `at` for w's gradient
    with torch.no_grad():
        call(at)
    assert bool((at != 0).any())
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    (at * w).sum().backward()
    assert torch.equal(w.grad, at)


@pytest.mark.parametrize("call", CALLS)
def test_inference_tensors(call):
    with torch.inference_mode():
        at = torch.zeros(2, 3, device="cuda")
        call(at)
        assert bool((at != 0).any())
