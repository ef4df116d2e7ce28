"""A network of detailed cells taught by a teacher's top logits, then answering in a closed loop.

Every learning tick the readout turns the cells' soma voltages into logits: a projection to
queries, keys and values, linear attention whose heads remember for different times, and a
projection to classes.  One training pass is

  capture_signals_cached   the network runs, its outputs and synaptic currents are kept
  Readout.forward          logits of every tick (linear_attention)
  distill_loss_grad        the loss against the teacher's top logits, and its gradient
  Readout.backward         gradients of the readout, and of the loss by the voltages
  replay_dw_from_cached_signals   from those the gradients of the synapses

and afterwards the network answers while it runs: fadvance, linear_attention_step, sample.

    python examples/teach_readout.py [--passes 8] [--cells 4]
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from heliox_amd import Sim, build_config, learn, readout  # noqa: E402

REST, RANGE = -65.0, 20.0        # mV; voltages enter the readout as (v - REST) / RANGE


class Readout:
    """Voltages (time, n_out) to logits (time, classes), with the gradients of both."""

    def __init__(self, n_out: int, classes: int, heads: int = 4, d: int = 16, seed: int = 0, device="cuda"):
        gen = torch.Generator().manual_seed(seed)
        weight = lambda n, m: (torch.randn(n, m, generator=gen) / n ** 0.5).to(device)  # noqa: E731
        self.heads, self.d = heads, d
        self.w_in, self.w_out = weight(n_out, 3 * heads * d), weight(heads * d, classes)
        # memories of 4 ticks to 256
        self.log_decay = -1.0 / (4.0 * 64.0 ** (torch.arange(heads, dtype=torch.float32) / max(heads - 1, 1))).to(device)

    def _qkv(self, x: torch.Tensor):
        return (x @ self.w_in).unflatten(-1, (3, self.heads, self.d)).unbind(-3)

    def forward(self, voltages: torch.Tensor) -> torch.Tensor:
        self.x = (voltages - REST) / RANGE
        self.qkv = [t[None] for t in self._qkv(self.x)]
        o, self.state = readout.linear_attention(*self.qkv, self.log_decay)
        self.o = o[0].flatten(1)
        return self.o @ self.w_out

    def backward(self, dlogits: torch.Tensor):
        """Gradients of w_in and w_out, and of the loss by the voltages of the last forward."""
        do = (dlogits @ self.w_out.t()).unflatten(-1, (self.heads, self.d))[None]
        dqkv = readout.linear_attention_grad(*self.qkv, self.log_decay, do)[:3]
        dy = torch.stack([t[0] for t in dqkv], dim=-3).flatten(-3)
        return self.x.t() @ dy, self.o.t() @ dlogits, dy @ self.w_in.t() / RANGE

    def start(self) -> torch.Tensor:
        return torch.zeros(1, self.heads, self.d, self.d, device=self.w_in.device)

    def step(self, voltages: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
        """Logits (1, classes) of one tick; state goes on in place."""
        q, k, v = self._qkv((voltages - REST) / RANGE)
        return readout.linear_attention_step(q, k, v, self.log_decay, state).flatten(1) @ self.w_out


class Network:
    """Cells of the second benchmark configuration, with what a capture and a replay need."""

    def __init__(self, cells: int, ticks: int, k_mul: int = 40):
        spec = build_config(2, cells, 1000.0)
        spec.netcons["ExpSyn"].weight = spec.netcons["ExpSyn"].weight * 20
        self.sim, self.ticks, self.k_mul, self.dt = Sim(), ticks, k_mul, spec.dt
        self.sim.load_model_from_spec(spec, add_monitors=False)
        nodes = spec.mechs["ExpSyn"].nodes
        n = nodes.size
        handle = self.sim.get_variable_handle
        self.somas = [handle("global", "v", i) for i in range(cells)]
        self.weights = [handle("ExpSyn", "weight", i) for i in range(n)]
        dest = np.arange(n, dtype=np.int32)
        cell = spec.cell_of_node()[nodes]
        self.capture = learn.CaptureSpec(
            output_v_handles=self.somas, tstop_ms=ticks * k_mul * self.dt, k_mul=k_mul, percise=False, v_init=REST,
            signals={"pure_i": learn.MappedSignal("pure_i", [handle("ExpSyn", "i", i) for i in range(n)], dest,
                                                  np.ones(n, np.float32))})
        # a synapse's current reaches the columns of its own cell, decaying over 8 ticks
        taps = np.exp(-np.arange(8)[::-1] / 3.0).astype(np.float32)
        same = (cell[:, None] == cell[None, :]).astype(np.float32)
        self.sim.set_dense_blocks_f32([np.ascontiguousarray(0.05 * same[:, :, None] * taps)])
        self.pre = np.full(n, -1, np.int32)
        self.outputs = np.array([np.flatnonzero(cell == c)[0] for c in range(cells)], np.int32)

    def run(self) -> torch.Tensor:
        """Voltages at the learning ticks, (ticks, cells)."""
        pack = learn.capture_signals_cached(self.sim, self.capture, total_steps=self.ticks * self.k_mul)
        return torch.from_numpy(pack.output_vs_tn[self.k_mul::self.k_mul].copy()).cuda()

    def learn(self, dvoltages: torch.Tensor, rate: float) -> np.ndarray:
        """The synapses' gradients from the loss's by the voltages; one step of descent."""
        dw = learn.replay_dw_from_cached_signals(
            self.sim, dLtdv_lr_ot=dvoltages.cpu().numpy(), poutput=self.outputs, pre_of_col=self.pre,
            dt_ms=self.dt * self.k_mul, percise=False)
        old = np.array(self.sim.get_variables_by_handles(self.weights))
        self.sim.set_variables_by_handles(self.weights, np.maximum(old - rate * dw, 0.0))
        return dw

    def tick(self) -> torch.Tensor:
        for _ in range(self.k_mul):
            self.sim.fadvance()
        return torch.tensor([self.sim.get_variables_by_handles(self.somas)], dtype=torch.float32, device="cuda")


def teacher_of(network: Network, voltages: torch.Tensor, classes: int, top: int):
    """What a trained network would have given for these ticks: its top logits, their places, and
    the logarithm of its whole sum."""
    logits = Readout(len(network.somas), classes, seed=7).forward(voltages) * 2.0
    best, at = torch.topk(logits, top, dim=1)
    return at.to(torch.int32), best, torch.logsumexp(logits, 1)


def teach(cells: int = 4, ticks: int = 100, classes: int = 50, passes: int = 8, rate: float = 0.1, say=print):
    network = Network(cells, ticks)
    student = Readout(cells, classes, seed=1)
    at, best, lse = teacher_of(network, network.run(), classes, top=5)
    weight = torch.full((ticks,), 1.0 / ticks, device="cuda")
    losses = []
    for n in range(passes):
        logits = student.forward(network.run())
        loss, dlogits = readout.distill_loss_grad(logits, at, best, teacher_lse=lse, weight=weight)
        dw_in, dw_out, dvoltages = student.backward(dlogits)
        dw = network.learn(dvoltages, rate=1e-6)
        student.w_in -= rate * dw_in
        student.w_out -= rate * dw_out
        losses.append(float(loss.mean()))
        say(f"pass {n}: loss {losses[-1]:.4f}, largest gradient of a synapse {np.abs(dw).max():.2e}")
    return network, student, losses


def answer(network: Network, student: Readout, ticks: int = 20, seed: int = 0):
    """The network runs and answers at every tick: tokens, and the logits that they came from."""
    u = torch.rand(ticks, generator=torch.Generator().manual_seed(seed)).cuda()
    network.sim.finitialize(REST)
    state, tokens, logits = student.start(), [], []
    for t in range(ticks):
        logits.append(student.step(network.tick(), state))
        tokens.append(readout.sample(logits[-1], u[t:t + 1], temperature=0.8, top_k=10, top_p=0.95)[0])
    return torch.cat(tokens), torch.cat(logits)


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--passes", type=int, default=8)
    ap.add_argument("--cells", type=int, default=4)
    args = ap.parse_args()
    network, student, _ = teach(cells=args.cells, passes=args.passes)
    print("answers:", answer(network, student)[0].tolist())


if __name__ == "__main__":
    main()
