"""The training operators and tensors that are more than memory: fake ones, wrapped ones, ones with a tangent, calls that are being traced."""
import subprocess
import sys

import pytest
import torch

from nano_nccl_b200 import ops

pytestmark = pytest.mark.gpu

# In a process of its own: what goes wrong here ends it.
WITHOUT_MEMORY = """
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from nano_nccl_b200 import ops
p, f, w = torch.arange(5, device="cuda"), ops.rotary_frequencies(64)[0], torch.ones(64, device="cuda")
kept, dy = ops.pack8(torch.ones(5, 64, device="cuda")), torch.ones(5, 8, device="cuda")
def calls(x):
    return [lambda: ops.pack8(x), lambda: ops.gelu8(x), lambda: ops.weight_grad8(x, kept), lambda: ops.rotary(x[:, None], None, p, f),
            lambda: ops.qk_norm_rotary(x[:, None], None, w, None, p, f)]
def refused(call):
    try:
        call()
    except (RuntimeError, ValueError):
        return
    raise SystemExit("not refused")
with FakeTensorMode(allow_non_fake_inputs=True):
    fake = torch.empty(5, 64, device="cuda")
for x in (fake, torch.nn.Parameter(fake)):
    for call in calls(x):
        refused(call)
for i in range(5):
    refused(lambda: torch.func.vmap(lambda x: calls(x)[i]())(torch.ones(2, 5, 64, device="cuda")))
    refused(lambda: torch.func.grad(lambda x: (calls(x)[i](), x.sum())[1])(torch.ones(5, 64, device="cuda")))
torch.cuda.synchronize()
print("alive", float(ops.gelu8(torch.zeros(1, device="cuda"))))
"""


def test_tensors_without_memory_of_their_own():
    run = subprocess.run([sys.executable, "-c", WITHOUT_MEMORY], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "alive 0.0" in run.stdout, run.stderr[-2000:] + run.stdout
