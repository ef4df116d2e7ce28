"""AdamW over as many tensors of one pair of types as a launch lists, and more; sizes around a wave's 512 and a workgroup's 2048."""
import pytest
import torch

from heliox_amd import readout
from test_gpu_readout_adamw import HOW, check_step

pytestmark = pytest.mark.gpu

SIZES = [1, 255, 256, 257, 511, 512, 513, 767, 1023, 1024, 1025, 2047, 2048, 2049, 4097]


def tensors(seed, count, dtype):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(SIZES[i * 7 % len(SIZES)], generator=gen).to(dtype).cuda() for i in range(count)]


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("count", [1, 63, 64, 65, 128, 130])
@pytest.mark.parametrize("kinds", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
def test_tensors_of_one_pair(bits, count, kinds):
    """Parameters, moments and scales of every tensor, after each of two steps."""
    params = tensors(0, count, kinds[0])
    state = readout.adamw_state(params, bits=bits)
    decays = [0.01 * (i % 5) for i in range(count)]
    for t in (1, 2):
        check_step(params, tensors(t, count, kinds[1]), state, t, {**HOW, "weight_decay": decays}, decays)


@pytest.mark.parametrize("bits", [8, 32])
def test_two_pairs_by_turns(bits):
    """65 of each of two pairs of types, by turns, empty tensors and missing gradients between them."""
    gen = torch.Generator().manual_seed(3)
    kinds = [torch.float32 if i % 2 else torch.bfloat16 for i in range(150)]
    sizes = [0 if i % 15 == 7 else SIZES[i % len(SIZES)] for i in range(150)]
    params = [torch.randn(n, generator=gen).to(k).cuda() for n, k in zip(sizes, kinds)]
    grads = [torch.randn(n, generator=gen).to(k).cuda() if i % 10 else None for i, (n, k) in enumerate(zip(sizes, kinds))]
    state, alone = readout.adamw_state(params, bits=bits), []
    for p, g in zip(params, grads):                             # each by itself
        one, its = p.clone(), readout.adamw_state([p], bits=bits)
        for _ in range(2):
            readout.adamw_step([one], [g], its, **HOW)
        alone.append((one, its))
    for _ in range(2):
        readout.adamw_step(params, grads, state, **HOW)
    torch.cuda.synchronize()
    for i, (one, its) in enumerate(alone):
        assert torch.equal(params[i], one), i
        at = slice(state.starts[i], state.starts[i] + -(-sizes[i] // 256) * 256)
        for name in ("m", "v"):
            assert torch.equal(getattr(state, name)[at].view(torch.uint8), getattr(its, name).view(torch.uint8)), i
        if bits == 8:
            blocks = slice(at.start // 256, at.stop // 256)
            assert torch.equal(state.m_scale[blocks], its.m_scale) and torch.equal(state.v_scale[blocks], its.v_scale)
