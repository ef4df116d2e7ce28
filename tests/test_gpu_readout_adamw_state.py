"""What an AdamW state does with tensors that are assigned to it, and when its own were changed."""
import copy
import io

import pytest
import torch

from heliox_amd import readout

pytestmark = pytest.mark.gpu

SIZES = [300, 5, 1000]


def tensors(seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(n, generator=gen).cuda() for n in SIZES]


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_a_checkpoint_is_assigned(bits, device):
    """It is copied: another state goes on as the saved one does, and the saved tensors stay."""
    params, grads = tensors(0), tensors(1)
    state = readout.adamw_state(params, bits=bits)
    for _ in range(3):
        readout.adamw_step(params, grads, state, lr=0.1)
    names = ("m", "v", "m_scale", "v_scale", "step")
    saved = {name: None if getattr(state, name) is None else getattr(state, name).clone().to(device) for name in names}
    kept = {name: None if x is None else x.clone() for name, x in saved.items()}
    again, other = [p.clone() for p in params], readout.adamw_state(params, bits=bits)
    at = other.m.data_ptr(), other.step.data_ptr()
    for name, x in saved.items():
        setattr(other, name, x)
    assert at == (other.m.data_ptr(), other.step.data_ptr()) and int(other.step) == 3
    readout.adamw_step(params, grads, state, lr=0.1)
    readout.adamw_step(again, grads, other, lr=0.1)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(params, again)) and int(other.step) == 4
    for name, x in saved.items():
        assert x is None or torch.equal(x.view(torch.uint8) if x.dtype.itemsize == 1 else x,
                                        kept[name].view(torch.uint8) if x.dtype.itemsize == 1 else kept[name])


def test_a_copy_counts_by_itself():
    params, grads = tensors(0), tensors(1)
    state = readout.adamw_state(params, bits=8)
    readout.adamw_step(params, grads, state, lr=0.1)
    other = copy.deepcopy(state)
    readout.adamw_step(params, grads, other, lr=0.1)
    assert int(state.step) == 1 and int(other.step) == 2
    state.step = 7
    readout.adamw_step(params, grads, state, lr=0.1)
    assert int(state.step) == 8


def test_a_saved_state_goes_on():
    params, grads = tensors(0), tensors(1)
    state, file = readout.adamw_state(params, bits=8), io.BytesIO()
    readout.adamw_step(params, grads, state, lr=0.1)
    torch.save(state, file)
    again = [p.clone() for p in params]
    other, host = (torch.load(io.BytesIO(file.getvalue()), weights_only=False, map_location=at) for at in (None, "cpu"))
    readout.adamw_step(params, grads, state, lr=0.1)
    readout.adamw_step(again, grads, other, lr=0.1)
    assert all(torch.equal(a, b) for a, b in zip(params, again)) and int(other.step) == 2
    with pytest.raises(ValueError, match="were changed"):       # on the CPU
        readout.adamw_step(again, grads, host, lr=0.1)


def test_assignments_are_refused():
    state, wide = readout.adamw_state(tensors(0), bits=8), readout.adamw_state(tensors(0))
    n = state.m.numel()
    for target, name, x, error, text in (
            (state, "m", torch.zeros(n), TypeError, "float8"), (wide, "m", torch.zeros(n, dtype=torch.float64), TypeError, "float32"),
            (wide, "m", torch.zeros(n - 1), ValueError, "shape"), (wide, "v", torch.zeros(n + 256), ValueError, "shape"),
            (wide, "v", torch.zeros(n, 1), ValueError, "shape"), (wide, "m", None, TypeError, "a tensor"),
            (wide, "m", [0.0] * n, TypeError, "a tensor"), (wide, "m_scale", torch.zeros(n // 256), TypeError, "None"),
            (state, "v_scale", None, TypeError, "a tensor"), (state, "m_scale", torch.zeros(n), ValueError, "shape"),
            (state, "step", torch.zeros(1), TypeError, "int64"), (state, "step", torch.zeros(2, dtype=torch.int64), TypeError, "one"),
            (state, "step", 1.0, TypeError, "whole"), (state, "step", 2 ** 70, ValueError, "large"),
            (state, "step", -1, ValueError, "at least 0")):
        with pytest.raises(error, match=text):
            setattr(target, name, x)
    assert all(not bool(s.m.float().any()) and int(s.step) == 0 for s in (state, wide))
    wide.m_scale = None


@pytest.mark.parametrize("name,change", [
    ("m", lambda x: setattr(x, "data", torch.zeros_like(x, device="cpu"))),
    ("v", lambda x: setattr(x, "data", x[:256].clone())),
    ("m_scale", lambda x: setattr(x, "data", torch.zeros(2 * x.numel(), device="cuda")[::2])),
    ("v_scale", lambda x: x.resize_(3))])
def test_a_state_whose_tensors_were_changed_is_refused(name, change):
    """Addresses that are none of the GPU's, or of too little memory, are not handed on."""
    params, grads = tensors(0), tensors(1)
    state = readout.adamw_state(params, bits=8)
    kept = [p.clone() for p in params]
    change(getattr(state, name))
    with pytest.raises(ValueError, match="were changed"):
        readout.adamw_step(params, grads, state, lr=0.1)
    assert all(torch.equal(a, b) for a, b in zip(params, kept)) and int(state.step) == 0


@pytest.mark.parametrize("bits,error", [(8.0, TypeError), ("8", TypeError), (None, TypeError), (16, ValueError), (2 ** 70, ValueError)])
def test_bits_are_whole_numbers(bits, error):
    with pytest.raises(error, match="bits"):
        readout.adamw_state(tensors(0), bits=bits)
