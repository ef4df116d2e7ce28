"""Settings of layer norm and the AdamW step that fp32 cannot hold are refused (no GPU)."""
import pytest
import torch

from heliox_amd import lib, readout
from test_readout_training import Tensors, error, norm

# over fp32's largest; an epsilon that is zero in fp32, and ones whose reciprocal is infinite there
TOO_LARGE, TOO_SMALL = 3.5e38, [1e-50, 1e-46, 1e-40, 1.17e-38]


def step(**change):
    lists = Tensors()
    return lib().hx_adamw_step(lists.record(moments=0, **change))


@pytest.mark.parametrize("change,text", [({"lr": TOO_LARGE}, "lr"), ({"lr": -TOO_LARGE}, "lr"), ({"scale": TOO_LARGE}, "grad_scale"),
                                         ({"eps": TOO_LARGE}, "eps"), *(({"eps": e}, "eps") for e in TOO_SMALL)])
def test_adamw(change, text):
    assert step(**change) == -1 and text in error()


@pytest.mark.parametrize("decay", [TOO_LARGE, -TOO_LARGE])
def test_adamw_decays(decay):
    lists = Tensors(decays=(1, decay))
    assert lib().hx_adamw_step(lists.record()) == -1 and "tensor 1: weight_decay" in error()


@pytest.mark.parametrize("eps", [TOO_LARGE, *TOO_SMALL])
@pytest.mark.parametrize("call", ["hx_layer_norm", "hx_layer_norm_grad", "hx_layer_norm_workspace"])
def test_layer_norm(call, eps):
    assert getattr(lib(), call)(norm(eps=eps)) == -1 and "eps" in error()


@pytest.mark.parametrize("eps", [0.0, 2.0 ** -126, 1e-12, 3e38])
def test_what_fits_goes_on(eps):
    assert lib().hx_layer_norm_workspace(norm(eps=eps)) > 0
    # (no room for moments: refused after the settings)
    assert step(eps=eps, lr=3e38, scale=-3e38) == -1 and "too few" in error()


@pytest.mark.parametrize("decay,error_type", [([0.1, 10 ** 400], ValueError), (10 ** 400, ValueError), ([0.1, "0.1"], TypeError),
                                              ([0.1, None], TypeError), ([0.1, torch.zeros(2)], TypeError), ((0.1,), ValueError)])
def test_decays_that_are_no_numbers(decay, error_type):
    with pytest.raises(error_type, match="weight_decay"):
        readout._decays(decay, 2)
