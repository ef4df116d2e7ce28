"""A network of detailed cells read out by a gated recurrence, which learns from rewards.

Every learning tick the readout turns the cells' soma voltages into logits: layer norm, a
projection to values and gates, the gated recurrence, a projection to classes.  One pass is

  capture_signals_cached   the network runs, its outputs and synaptic currents are kept
  Readout.forward          logits of every tick (layer_norm, gated_recurrence)
  sample, token_logprobs   an answer for every tick, its log probability, the logits' entropy
  token_logprobs_grad      the gradient of what the answers earned, and of a term for the entropy
  Readout.backward         gradients of the readout, and of the loss by the voltages
  adamw_step               the readout's parameters, all at once, moments in 8 bits
  replay_dw_from_cached_signals   the gradients of the synapses

and afterwards the network answers while it runs: fadvance, gated_recurrence_step, sample, with the
alternatives that it did not take.

    python examples/recurrent_readout.py [--passes 8] [--cells 4]
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [HERE, os.path.dirname(HERE)]

from heliox_amd import readout  # noqa: E402
from teach_readout import REST, Network  # noqa: E402


class Readout:
    """Voltages (time, n_out) to logits (time, classes), with the gradients of both."""

    NAMES = ("norm_weight", "norm_bias", "w_in", "w_out")

    def __init__(self, n_out: int, classes: int, channels: int = 64, seed: int = 0, bits: int = 8, device="cuda"):
        gen = torch.Generator().manual_seed(seed)
        weight = lambda n, m: (torch.randn(n, m, generator=gen) / n ** 0.5).to(device)  # noqa: E731
        self.channels = channels
        self.norm_weight, self.norm_bias = torch.ones(n_out, device=device), torch.zeros(n_out, device=device)
        self.w_in, self.w_out = weight(n_out, 2 * channels), weight(channels, classes)
        # channels remember for 4 ticks to 256
        self.keep = torch.log(4.0 * 64.0 ** (torch.arange(channels) / max(channels - 1, 1)) - 1.0).to(device)
        self.state = readout.adamw_state(self.parameters(), bits=bits)

    def parameters(self) -> list:
        return [getattr(self, name) for name in self.NAMES]

    def _values_and_gates(self, n: torch.Tensor):
        value, gate = (n @ self.w_in).split(self.channels, dim=-1)
        return value, gate + self.keep

    def forward(self, voltages: torch.Tensor) -> torch.Tensor:
        self.v = voltages
        self.n, self.mean, self.rstd = readout.layer_norm(voltages, self.norm_weight, self.norm_bias)
        self.value, self.gate = (t[None] for t in self._values_and_gates(self.n))
        o, _ = readout.gated_recurrence(self.value, self.gate)
        self.o = o[0]
        return self.o @ self.w_out

    def backward(self, dlogits: torch.Tensor):
        """Gradients of the parameters, and of the loss by the voltages of the last forward."""
        do = (dlogits @ self.w_out.t())[None]
        dvalue, dgate, _ = readout.gated_recurrence_grad(self.value, self.gate, do)
        dy = torch.cat([dvalue[0], dgate[0]], dim=-1)
        dv, dweight, dbias = readout.layer_norm_grad(self.v, self.norm_weight, self.mean, self.rstd, dy @ self.w_in.t())
        return [dweight, dbias, self.n.t() @ dy, self.o.t() @ dlogits], dv

    def learn(self, grads: list, rate: float) -> None:
        # matrices decay, vectors do not
        readout.adamw_step(self.parameters(), grads, self.state, lr=rate, weight_decay=[0.0, 0.0, 0.01, 0.01])

    def start(self) -> torch.Tensor:
        return torch.zeros(1, self.channels, device=self.w_in.device)

    def step(self, voltages: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
        """Logits (1, classes) of one tick; state goes on in place."""
        n, _, _ = readout.layer_norm(voltages, self.norm_weight, self.norm_bias)
        return readout.gated_recurrence_step(*self._values_and_gates(n), state) @ self.w_out


def reward_of(ticks: int, classes: int, seed: int = 7) -> torch.Tensor:
    """What each class earns at each tick: one of them 1 for 10 ticks, then another."""
    right = torch.randint(classes, (ticks // 10 + 1,), generator=torch.Generator().manual_seed(seed))
    earned = torch.zeros(ticks, classes)
    earned[torch.arange(ticks), right.repeat_interleave(10)[:ticks]] = 1.0
    return earned.cuda()


def gradient(logits: torch.Tensor, token: torch.Tensor, earned: torch.Tensor, entropy_weight: float):
    """The loss -mean(advantage log q_token + entropy_weight entropy) by the logits, and its terms."""
    scored = readout.token_logprobs(logits, token)
    ticks = len(token)
    gain = earned.gather(1, token[:, None])[:, 0]
    dlogprob = -(gain - gain.mean()) / ticks
    dentropy = torch.full_like(dlogprob, -entropy_weight / ticks)
    return readout.token_logprobs_grad(logits, token, scored, dlogprob, dentropy), gain, scored.entropy


def train(cells: int = 4, ticks: int = 100, classes: int = 8, passes: int = 8, rate: float = 0.02, say=print):
    network = Network(cells, ticks)
    student = Readout(cells, classes, seed=1)
    earned = reward_of(ticks, classes)
    gen = torch.Generator().manual_seed(3)
    history = []
    for n in range(passes):
        logits = student.forward(network.run())
        token, _ = readout.sample(logits, torch.rand(ticks, generator=gen).cuda())
        dlogits, gain, entropy = gradient(logits, token, earned, entropy_weight=0.01)
        grads, dvoltages = student.backward(dlogits)
        student.learn(grads, rate)
        dw = network.learn(dvoltages, rate=1e-6)
        history.append((float(gain.mean()), float(entropy.mean()), float(np.abs(dw).max())))
        say(f"pass {n}: earned {history[-1][0]:.3f}, entropy {history[-1][1]:.3f}, "
            f"largest gradient of a synapse {history[-1][2]:.2e}")
    return network, student, history


def answer(network: Network, student: Readout, ticks: int = 20, seed: int = 0):
    """The network runs and answers at every tick: tokens, their log probabilities with the three
    likeliest alternatives, and the logits that they came from."""
    u = torch.rand(ticks, generator=torch.Generator().manual_seed(seed)).cuda()
    network.sim.finitialize(REST)
    state, tokens, scored, logits = student.start(), [], [], []
    for t in range(ticks):
        logits.append(student.step(network.tick(), state))
        tokens.append(readout.sample(logits[-1], u[t:t + 1])[0])
        scored.append(readout.token_logprobs(logits[-1], tokens[-1], top=3))
    return torch.cat(tokens), scored, torch.cat(logits)


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--passes", type=int, default=8)
    ap.add_argument("--cells", type=int, default=4)
    args = ap.parse_args()
    network, student, _ = train(cells=args.cells, passes=args.passes)
    tokens, scored, _ = answer(network, student)
    for token, s in zip(tokens.tolist(), scored):
        others = ", ".join(f"{i}: {p:.2f}" for i, p in zip(s.top_index[0].tolist(), s.top_logprob[0].tolist()))
        print(f"answer {token} at {float(s.logprob):.2f}; likeliest {others}")


if __name__ == "__main__":
    main()
