"""Refusals of layer norm, the gated recurrence, token log probabilities and the AdamW step, in Python
and at the C entry points (no GPU).  Pointers are only compared: every call ends before a launch."""
import os
import shutil
import subprocess
from array import array

import pytest
import torch

from heliox_amd import lib, readout

AT = 1 << 40


def error():
    return lib().hx_readout_error().decode()


def norm(type=0, weight_type=0, rows=5, width=8, x=AT, eps=1e-5, y=AT, stats=AT, dy=AT, dx=AT, dw=AT, db=AT, space=0, size=0):
    return readout._NORM.pack(type, weight_type, rows, width, x, width, 0, 0, eps, y, width, stats, stats, dy, width, dx,
                              width, dw, db, space, size, 0)


@pytest.mark.parametrize("call", ["hx_layer_norm", "hx_layer_norm_grad", "hx_layer_norm_workspace"])
@pytest.mark.parametrize("change,text", [
    ({"type": 3}, "type"), ({"weight_type": -1}, "type"), ({"rows": -1}, "rows"), ({"rows": 2 ** 31}, "rows"),
    ({"width": 0}, "width"), ({"width": 2 ** 24 + 1}, "width"), ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"),
    ({"eps": float("inf")}, "eps"), ({"dw": 0}, "together"), ({"db": 0}, "together")])
def test_norm_is_refused(call, change, text):
    assert getattr(lib(), call)(norm(**change)) == -1
    assert call in error() and text in error()


def test_norm_missing_pointers_and_workspace():
    L = lib()
    for name in ("x", "y", "stats"):
        assert L.hx_layer_norm(norm(**{name: 0})) == -1 and "missing" in error()
    for name in ("x", "dy", "dx", "stats"):
        assert L.hx_layer_norm_grad(norm(**{name: 0})) == -1 and "missing" in error()
    need = L.hx_layer_norm_workspace(norm())
    assert need > 0
    for space, size, text in ((0, need, "hold"), (4096, need - 1, "hold"), (4096, -1, "hold"), (4104, need, "16 bytes")):
        assert L.hx_layer_norm_grad(norm(space=space, size=size)) == -1 and text in error()
    assert L.hx_layer_norm(None) == L.hx_layer_norm_grad(None) == L.hx_layer_norm_workspace(None) == -1
    assert L.hx_layer_norm(norm(rows=0, x=0, y=0)) == 0
    assert L.hx_layer_norm_grad(norm(rows=0, dw=0, db=0)) == 0
    assert L.hx_layer_norm_workspace(norm(dw=0, db=0)) == 0


def recurrence(type=0, batch=2, time=5, channels=8, x=AT, gate=AT, initial=0, o=AT, end=0, do=AT, dend=0, dx=AT, dgate=AT,
               dinitial=0, state=AT, slots=0, n_slots=0, space=0, size=0):
    return readout._RECURRENCE.pack(type, batch, time, channels, x, gate, 0, 0, 0, 0, initial, 0, o, 0, 0, end, do, 0, 0, dend,
                                    dx, dgate, dinitial, state, slots, n_slots, space, size, 0)


@pytest.mark.parametrize("call", ["hx_gated_recurrence", "hx_gated_recurrence_grad", "hx_gated_recurrence_step"])
@pytest.mark.parametrize("change,text", [
    ({"type": 5}, "type"), ({"batch": -1}, "negative"), ({"time": -1}, "negative"), ({"channels": 0}, "channels"),
    ({"batch": 2 ** 28}, "2^31"), ({"batch": 2 ** 62}, "2^31"), ({"channels": 2 ** 40, "batch": 0}, "2^31"),
    ({"channels": 2 ** 30 + 1, "batch": 1}, "2^30"),
    ({"time": 2 ** 30 + 1}, "2^30")])
def test_recurrence_sizes_are_refused(call, change, text):
    assert getattr(lib(), call)(recurrence(**change)) == -1
    assert call in error() and text in error()


def test_recurrence_missing_pointers():
    L = lib()
    for call, names in (("hx_gated_recurrence", ("x", "gate", "o")), ("hx_gated_recurrence_grad", ("x", "gate", "do", "dx", "dgate")),
                        ("hx_gated_recurrence_step", ("x", "gate", "o", "state"))):
        one = dict(time=1, n_slots=2) if "step" in call else {}
        for name in names:
            assert getattr(L, call)(recurrence(**one, **{name: 0})) == -1 and "missing" in error()
        assert getattr(L, call)(None) == -1
        assert getattr(L, call)(recurrence(**{**one, "batch": 0})) == 0
    assert L.hx_gated_recurrence_step(recurrence()) == -1 and "time" in error()
    assert L.hx_gated_recurrence_step(recurrence(time=1, n_slots=1)) == -1 and "only 1 states" in error()
    assert L.hx_gated_recurrence_step(recurrence(time=1, n_slots=-1)) == -1 and "negative" in error()


@pytest.mark.parametrize("grad", [0, 1])
def test_recurrence_workspace(grad):
    L, call = lib(), "hx_gated_recurrence_grad" if grad else "hx_gated_recurrence"
    assert L.hx_gated_recurrence_workspace(recurrence(channels=0), grad) == -1
    assert L.hx_gated_recurrence_workspace(recurrence(), grad) == 0
    need = L.hx_gated_recurrence_workspace(recurrence(time=5000), grad)
    assert 0 < need < L.hx_gated_recurrence_workspace(recurrence(time=50000), grad)
    for space, size, text in ((0, need, "hold"), (4096, need - 1, "hold"), (4104, need, "16 bytes")):
        assert getattr(L, call)(recurrence(time=5000, space=space, size=size)) == -1 and text in error()


@pytest.mark.parametrize("call,out,into", [("hx_gated_recurrence", "end", "initial"),
                                           ("hx_gated_recurrence_grad", "dinitial", "initial"),
                                           ("hx_gated_recurrence_grad", "dinitial", "dend")])
def test_states_written_over_those_read_are_refused(call, out, into):
    size = 4 * 2 * 8
    for apart, refused in ((0, True), (size - 4, True), (4 - size, True), (size, False), (-size, False)):
        assert getattr(lib(), call)(recurrence(time=5000, **{into: 1 << 20, out: (1 << 20) + apart})) == -1
        assert ("overlaps" in error()) == refused and ("workspace" in error()) != refused


def logprob(type=0, bits=64, rows=4, vocab=10, top=3, logits=AT, stride=10, tokens=AT, tau=1.0, out=AT, entropy=AT, stats=AT,
            tops=AT, grad=1 << 41, grad_stride=10, space=0, size=0):
    return readout._LOGPROB.pack(type, bits, rows, vocab, top, logits, stride, tokens, tau, out, entropy, stats, tops, tops, 0, 0,
                                 grad, grad_stride, space, size, 0)


@pytest.mark.parametrize("call", ["hx_token_logprobs", "hx_token_logprobs_grad", "hx_token_logprobs_workspace"])
@pytest.mark.parametrize("change,text", [
    ({"type": 9}, "type"), ({"bits": 16}, "bits"), ({"rows": -1}, "rows"), ({"rows": 2 ** 21 + 1}, "rows"), ({"vocab": 0}, "vocab"),
    ({"vocab": 2 ** 22 + 1}, "vocab"), ({"top": -1}, "top"), ({"top": 11}, "top"), ({"top": 257, "vocab": 1000}, "top"),
    ({"tau": 0.0}, "temperature"), ({"tau": -1.0}, "temperature"), ({"tau": float("nan")}, "temperature"),
    ({"tau": 2.0 ** -127}, "temperature"), ({"tau": 2.0 ** 127}, "temperature")])
def test_logprobs_are_refused(call, change, text):
    assert getattr(lib(), call)(logprob(**change)) == -1
    assert call in error() and text in error()


def test_logprobs_missing_pointers_and_workspace():
    L = lib()
    for name in ("logits", "tokens", "out", "entropy", "stats", "tops"):
        assert L.hx_token_logprobs(logprob(**{name: 0})) == -1 and "missing" in error()
    for name in ("logits", "tokens", "entropy", "stats", "grad"):
        assert L.hx_token_logprobs_grad(logprob(**{name: 0})) == -1 and "missing" in error()
    long = dict(rows=1, vocab=200000)
    need = L.hx_token_logprobs_workspace(logprob(**long))
    assert need > 0
    for space, size, text in ((0, need, "hold"), (4096, need - 1, "hold"), (4104, need, "16 bytes")):
        assert L.hx_token_logprobs(logprob(**long, space=space, size=size)) == -1 and text in error()
    assert L.hx_token_logprobs(None) == L.hx_token_logprobs_grad(None) == -1
    assert L.hx_token_logprobs(logprob(rows=0)) == L.hx_token_logprobs_grad(logprob(rows=0)) == 0


@pytest.mark.parametrize("kind,size", [(0, 4), (2, 2)])
@pytest.mark.parametrize("apart,stride,text", [(0, 0, "each other"), (500, 9, "each other"), (1, 10, "without being"),
                                               (-39, 10, "without being"), (0, 20, "without being"), (10, 30, "without being")])
def test_a_gradient_that_overlaps_is_refused(kind, size, apart, stride, text):
    at = 1 << 20
    assert lib().hx_token_logprobs_grad(logprob(type=kind, logits=at, grad=at + apart * size, grad_stride=stride)) == -1
    assert text in error()


class Tensors:
    """The lists of an AdamW call, kept for as long as their addresses are used."""

    def __init__(self, count=2, **change):
        self.lists = dict(types=array("q", [0] * count), grads_types=array("q", [2] * count),
                          params=array("Q", [AT + i * 4096 for i in range(count)]),
                          grads=array("Q", [2 * AT + i * 4096 for i in range(count)]), elements=array("q", [300] * count),
                          starts=array("q", [512 * i for i in range(count)]), decays=array("d", [0.1] * count))
        for name, (i, value) in change.items():
            self.lists[name][i] = value
        self.count = count

    def record(self, bits=32, m=AT, v=AT, scales=0, moments=1024, lr=0.1, beta1=0.9, beta2=0.99, eps=1e-8, scale=1.0, step=AT,
               count=None):
        return readout._ADAMW.pack(bits, self.count if count is None else count, *[a.buffer_info()[0] for a in self.lists.values()],
                                   m, v, scales, scales, moments, lr, beta1, beta2, eps, scale, 0, 0, step, 0)


@pytest.mark.parametrize("change,text", [
    ({"bits": 16}, "bits"), ({"count": -1}, "count"), ({"count": 2 ** 21}, "count"), ({"beta1": 1.0}, "beta1"),
    ({"beta2": -0.1}, "beta1"), ({"beta2": float("nan")}, "beta1"), ({"eps": -1.0}, "eps"), ({"eps": float("inf")}, "eps"),
    ({"lr": float("nan")}, "lr"), ({"scale": float("inf")}, "grad_scale"), ({"step": 0}, "step"), ({"m": 0}, "missing"),
    ({"v": 0}, "missing"), ({"bits": 8}, "scales"), ({"m": AT + 8}, "16 bytes"), ({"step": AT + 8}, "16 bytes"),
    ({"moments": -1}, "missing"), ({"moments": 1000}, "too few")])
def test_adamw_is_refused(change, text):
    lists = Tensors()
    assert lib().hx_adamw_step(lists.record(**change)) == -1
    assert "hx_adamw_step" in error() and text in error()


@pytest.mark.parametrize("change,text", [
    ({"types": (1, 3)}, "tensor 1: type"), ({"grads_types": (0, -1)}, "tensor 0: type"), ({"elements": (1, -1)}, "elements"),
    ({"elements": (0, 2 ** 35)}, "elements"), ({"elements": (0, 600)}, "after those before"), ({"starts": (1, 700)}, "multiples of 256"),
    ({"starts": (1, 256)}, "after those before"), ({"starts": (0, -256)}, "after those before"), ({"elements": (1, 600)}, "too few"),
    ({"params": (1, 0)}, "missing"), ({"grads": (0, 0)}, "missing"), ({"decays": (0, float("nan"))}, "weight_decay"),
    ({"params": (1, AT + 1196)}, "overlap"), ({"params": (1, AT - 1196)}, "overlap"), ({"grads": (0, AT + 600)}, "overlap"),
    ({"grads": (1, AT - 596)}, "overlap")])
def test_adamw_tensors_are_refused(change, text):
    lists = Tensors(**change)
    assert lib().hx_adamw_step(lists.record()) == -1
    assert text in error()
    assert lib().hx_adamw_step(None) == -1


def test_python_refuses_tensors_off_the_gpu():
    x = torch.zeros(2, 3, 8)
    for call in (lambda: readout.layer_norm(x), lambda: readout.layer_norm_grad(x, None, x[..., 0], x[..., 0], x),
                 lambda: readout.gated_recurrence(x, x), lambda: readout.gated_recurrence_grad(x, x, x),
                 lambda: readout.gated_recurrence_step(x[0], x[0], torch.zeros(3, 8)),
                 lambda: readout.token_logprobs(x[0], torch.zeros(3, dtype=torch.int64)),
                 lambda: readout.token_logprobs_grad(x[0], torch.zeros(3, dtype=torch.int64), None, None),
                 lambda: readout.adamw_state([x])):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for call in (lambda: readout.layer_norm([1.0]), lambda: readout.gated_recurrence(None, None), lambda: readout.adamw_state([None]),
                 lambda: readout.token_logprobs([[1.0]], None), lambda: readout.adamw_step([x], [x], None, lr=0.1)):
        with pytest.raises(TypeError):
            call()


def test_records_are_as_long_as_the_header_says(tmp_path):
    cc = shutil.which("g++") or shutil.which("c++")
    if cc is None:
        pytest.skip("no host compiler")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (tmp_path / "s.cpp").write_text('#include "heliox.h"\n#include <cstdio>\nint main() { printf("%zu %zu %zu %zu", '
                                    "sizeof(hx_norm_args), sizeof(hx_recurrence_args), sizeof(hx_logprob_args), "
                                    "sizeof(hx_adamw_args)); }\n")
    subprocess.run([cc, "-I", os.path.join(root, "include"), str(tmp_path / "s.cpp"), "-o", str(tmp_path / "s")], check=True)
    got = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout
    assert got.split() == [str(r.size) for r in (readout._NORM, readout._RECURRENCE, readout._LOGPROB, readout._ADAMW)]
