"""What a call does where its launches fail: the error comes back, and nothing else is touched (no GPU)."""
import subprocess
import sys

import pytest
import torch

STEP = """
import sys
sys.path[:0] = {path!r}
from heliox_amd import lib
from test_readout_training import Tensors, error
for count in (1, 64, 65, 66, 128, 300, 5000):
    print(count, flush=True)
    lists = Tensors(count)
    for i in range(count):
        lists.lists["types"][i] = i % {kinds}
    assert lib().hx_adamw_step(lists.record(moments=512 * count)) == -1
    assert error().startswith("hx_adamw_step: "), error()
"""


@pytest.mark.parametrize("kinds", [1, 3])
def test_adamw_of_more_tensors_than_a_launch_lists(kinds):
    """Without a device every launch fails.  (In a process of its own: the lists' addresses are none.)"""
    if torch.cuda.device_count():
        pytest.skip("launches do not fail where there is a GPU")
    code = STEP.format(path=sys.path[:], kinds=kinds)
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, (done.returncode, done.stdout[-20:], done.stderr[-2000:])
