"""Refusals of the readout operators, in Python and at the C entry points (no GPU)."""
import pytest
import torch

from heliox_amd import lib, readout

GOOD = dict(type=2, batch=2, time=5, heads=4, q_heads=4, k_heads=2, v_heads=1, dk=16, dv=24)


def attention(scale=1.0, n_slots=0, **sizes):
    s = {**GOOD, **sizes}
    return readout._ATTENTION.pack(*(s[n] for n in GOOD), 0, 0, 0, *[0] * 9, 0, 0, 0, scale, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0,
                                   0, 0, 0, 0, 0, 0, n_slots, 0, 0, 0)


def error():
    return lib().hx_readout_error().decode()


@pytest.mark.parametrize("change,text", [
    ({"type": 3}, "type"), ({"batch": -1}, "negative"), ({"time": -1}, "negative"), ({"heads": 0}, "heads"),
    ({"k_heads": 3}, "multiple"), ({"q_heads": 0}, "multiple"), ({"v_heads": 8}, "multiple"), ({"dk": 0}, "dk"),
    ({"dk": 257}, "dk"), ({"dv": 300}, "dv"), ({"scale": float("nan")}, "scale"), ({"batch": 2 ** 20}, "2^20"),
    ({"batch": 2 ** 62}, "2^20"), ({"time": 2 ** 40}, "2^30")])
@pytest.mark.parametrize("call", ["hx_linear_attention", "hx_linear_attention_grad", "hx_linear_attention_step"])
def test_attention_sizes_are_refused(call, change, text):
    assert getattr(lib(), call)(attention(**change)) == -1
    assert call in error() and text in error()


@pytest.mark.parametrize("call", ["hx_linear_attention", "hx_linear_attention_grad"])
def test_attention_missing_pointers_are_refused(call):
    assert getattr(lib(), call)(attention()) == -1
    assert "missing" in error()
    assert getattr(lib(), call)(None) == -1
    assert getattr(lib(), call)(attention(batch=0)) == 0


def test_step_is_refused():
    L = lib()
    assert L.hx_linear_attention_step(attention(time=5)) == -1 and "time" in error()
    assert L.hx_linear_attention_step(attention(time=1, n_slots=1)) == -1 and "states" in error()
    assert L.hx_linear_attention_step(attention(time=1, n_slots=2)) == -1 and "missing" in error()
    assert L.hx_linear_attention_step(attention(time=1, batch=0)) == 0


def test_workspace_grows_with_the_problem():
    L = lib()
    assert L.hx_linear_attention_workspace(attention(dk=999), 0) == -1
    small, large = (L.hx_linear_attention_workspace(attention(time=t), 1) for t in (5, 5000))
    assert 0 <= small <= large


def distill(type=0, teacher_type=0, bits=32, rows=2, vocab=9, top=3, temperature=1.0):
    return readout._DISTILL.pack(type, teacher_type, bits, rows, vocab, top, 0, 0, 0, 0, 0, 0, 0, 0, temperature, 0, 0,
                                 0, 0)


@pytest.mark.parametrize("change,text", [
    ({"type": 7}, "type"), ({"teacher_type": -1}, "type"), ({"bits": 16}, "bits"), ({"rows": -1}, "rows"), ({"rows": 2 ** 21 + 1}, "rows"),
    ({"vocab": 0}, "vocab"), ({"vocab": 2 ** 20 + 1}, "vocab"), ({"top": 2049}, "top"), ({"top": -1}, "top"),
    ({"temperature": 0.0}, "temperature"), ({"temperature": float("inf")}, "temperature"),
    ({"temperature": float("nan")}, "temperature"), ({}, "missing")])
def test_distill_is_refused(change, text):
    assert lib().hx_distill_loss(distill(**change)) == -1
    assert text in error()


@pytest.mark.parametrize("sizes,text", [((9, 1, 5), "type"), ((0, -1, 5), "rows"), ((0, 2 ** 21 + 1, 5), "rows"), ((0, 1, 0), "vocab"),
                                        ((0, 1, 2 ** 22 + 1), "vocab"), ((0, 1, 5), "missing")])
def test_sample_is_refused(sizes, text):
    record = readout._SAMPLE.pack(*sizes, 0, 0, 0, 0, 0, 0, 0, 1.0, 1.0, 0.0, 0, 0, 0, 0)
    assert lib().hx_sample(record) == -1
    assert text in error()


def test_empty_problems_need_no_gpu():
    assert lib().hx_distill_loss(distill(rows=0)) == 0
    assert lib().hx_sample(readout._SAMPLE.pack(0, 0, 5, 0, 0, 0, 0, 0, 0, 0, 1.0, 1.0, 0.0, 0, 0, 0, 0)) == 0


def test_python_refuses_tensors_off_the_gpu():
    x = torch.zeros(2, 3, 4, 8)
    with pytest.raises(ValueError, match="GPU"):
        readout.linear_attention(x, x, x, torch.zeros(4))
    with pytest.raises(ValueError, match="GPU"):
        readout.linear_attention_grad(x, x, x, torch.zeros(4), x)
    with pytest.raises(ValueError, match="GPU"):
        readout.linear_attention_step(x[:, 0], x[:, 0], x[:, 0], torch.zeros(4), torch.zeros(2, 4, 8, 8))
    with pytest.raises(ValueError, match="GPU"):
        readout.sample(x[0, 0], torch.zeros(4))
    with pytest.raises(ValueError, match="GPU"):
        readout.distill_loss_grad(x[0, 0], torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, 1))
    with pytest.raises(TypeError, match="tensor"):
        readout.sample([[1.0]], torch.zeros(1))


def test_records_are_as_long_as_the_header_says(tmp_path):
    import os
    import shutil
    import subprocess

    cc = shutil.which("g++") or shutil.which("c++")
    if cc is None:
        pytest.skip("no host compiler")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (tmp_path / "s.cpp").write_text('#include "heliox.h"\n#include <cstdio>\nint main() { printf("%zu %zu %zu", '
                                    "sizeof(hx_attention_args), sizeof(hx_distill_args), sizeof(hx_sample_args)); }\n")
    subprocess.run([cc, "-I", os.path.join(root, "include"), str(tmp_path / "s.cpp"), "-o", str(tmp_path / "s")],
                   check=True)
    got = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout
    assert got.split() == [str(r.size) for r in (readout._ATTENTION, readout._DISTILL, readout._SAMPLE)]


def test_a_workspace_that_does_not_fit_is_refused():
    """Pointers are only compared here: the call ends before anything is launched."""
    long = dict(GOOD, batch=1, time=5000)
    need = lib().hx_linear_attention_workspace(attention(**long), 0)
    assert need > 0
    fields = list(readout._ATTENTION.unpack(attention(**long)))
    for i in (9, 10, 11, 21, 25):       # q, k, v, log_decay, o
        fields[i] = 4096
    for space, size in ((0, need), (4096, need - 1), (4096, -1)):
        fields[-3:-1] = space, size
        assert lib().hx_linear_attention(readout._ATTENTION.pack(*fields)) == -1
        assert "workspace" in error()
    fields[-3:-1] = 4104, need
    assert lib().hx_linear_attention(readout._ATTENTION.pack(*fields)) == -1 and "16 bytes" in error()


@pytest.mark.parametrize("temperature", [2.0 ** -127, 1e-300, 2.0 ** 127, 1e300, -1.0])
def test_temperatures_that_fp32_cannot_hold_are_refused(temperature):
    """Its reciprocal, or the temperature itself, would be infinite in the kernel and the result NaN."""
    assert lib().hx_distill_loss(distill(temperature=temperature)) == -1
    assert "temperature" in error()


@pytest.mark.parametrize("temperature", [2.0 ** -126, 2.0 ** 126])
def test_temperatures_at_the_ends_are_taken(temperature):
    assert lib().hx_distill_loss(distill(rows=0, temperature=temperature)) == 0


@pytest.mark.parametrize("call,out,inp", [("hx_linear_attention", 29, 22), ("hx_linear_attention_grad", 38, 22),
                                          ("hx_linear_attention_grad", 38, 34)])
def test_states_written_over_those_read_are_refused(call, out, inp):
    """Pointers are only compared here: the call ends before anything is launched (no workspace)."""
    long = dict(GOOD, batch=1, time=5000)
    fields = list(readout._ATTENTION.unpack(attention(**long)))
    for i in (9, 10, 11, 21, 25, 30, 35, 36, 37):       # q, k, v, log_decay, o, grad_o, grad_q, grad_k, grad_v
        fields[i] = 1 << 40
    size = 4 * 4 * 16 * 24
    for apart, refused in ((0, True), (size - 4, True), (4 - size, True), (size, False), (-size, False)):
        fields[inp], fields[out] = 1 << 20, (1 << 20) + apart
        assert getattr(lib(), call)(readout._ATTENTION.pack(*fields)) == -1
        assert ("overlaps" in error()) == refused and ("workspace" in error()) != refused


@pytest.mark.parametrize("kind,size", [(0, 4), (1, 2)])
@pytest.mark.parametrize("rows,vocab,apart,logits_stride,grad_stride,text", [
    (4, 10, 0, 10, 0, "each other"),        # an expanded row
    (4, 10, 500, 10, 9, "each other"),
    (4, 10, 500, 10, -9, "each other"),
    (4, 10, 1, 10, 10, "without being"),    # one element further
    (4, 10, -39, 10, 10, "without being"),
    (4, 10, 0, 10, 20, "without being"),    # the same start, other rows
    (4, 10, 10, 20, 30, "without being"),
    (4, 10, 9, 20, 20, "without being"),
    (4, 10, 0, 0, 10, "without being"),
    (1, 10, 9, 0, 0, "without being"),
    (4, 10, -30, -10, 10, "without being")])
def test_a_gradient_that_overlaps_is_refused(kind, size, rows, vocab, apart, logits_stride, grad_stride, text):
    """Pointers are only compared here: the call ends before anything is launched."""
    at = 1 << 20
    record = readout._DISTILL.pack(kind, 0, 32, rows, vocab, 0, at, logits_stride, 0, 0, 0, 0, 0, 0, 1.0, 1 << 30,
                                   at + apart * size, grad_stride, 0)
    assert lib().hx_distill_loss(record) == -1
    assert text in error()
