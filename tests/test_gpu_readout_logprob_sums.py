"""Log probabilities of long rows whose logits are alike: thousands of equal terms a thread, whose roundings are alike too."""
import math

import pytest
import torch

from heliox_amd import readout

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24


@pytest.mark.parametrize("rows,vocab,dtype", [(512, 1 << 19, torch.float32), (512, 1 << 19, torch.float16), (600, 700_001, torch.bfloat16),
                                              (512, 1 << 22, torch.float16), (3, 1 << 22, torch.float32)])
@pytest.mark.parametrize("less,tau", [(0.6875, 1.0), (1.125, 1.5), (3.25, 40.0)])
@pytest.mark.parametrize("top", [0, 3])
def test_one_logit_above_equal_ones(rows, vocab, dtype, less, tau, top):
    """log z = log(1 + (n - 1) e^-d), d = less / tau, the entropy log z - sum q log.  A weight takes its argument's two
    roundings and the exponential's unit, 2 d + 2 halves; 8 of them and 4 such sums are added in fp32, at most 10
    more, what follows in 64 bits; results are rounded once.  The terms of s are d times as large, with two more each."""
    x = torch.full((rows, vocab), 2.0 - less, dtype=dtype, device="cuda")
    hot = torch.arange(rows, device="cuda") * 977 % vocab
    x[torch.arange(rows, device="cuda"), hot] = 2.0
    tokens = hot.clone()
    tokens[1::2] = (hot[1::2] + 1) % vocab
    got = readout.token_logprobs(x, tokens, temperature=tau, top=top)
    torch.cuda.synchronize()
    d = less / tau
    z = 1 + (vocab - 1) * math.exp(-d)
    logz, entropy = math.log(z), math.log(z) + (vocab - 1) * d * math.exp(-d) / z
    halves = 12 + 2 * d
    near = lambda t, want, more=0.0: float((t.double() - want).abs().max()) <= F32 * (halves + more + 2 * abs(want))  # noqa: E731
    assert near(got.stats[:, 1], logz)
    assert near(got.logprob[0::2], -logz) and near(got.logprob[1::2], -logz - d)
    assert near(got.entropy, entropy, d * (2 * halves + 2))
    if top:
        assert torch.equal(got.top_index[:, 0], hot) and near(got.top_logprob[:, 0], -logz) and near(got.top_logprob[:, 1:], -logz - d)
    assert bool((got.stats[:, 0] == 2.0).all())
    del x, got
    torch.cuda.empty_cache()
