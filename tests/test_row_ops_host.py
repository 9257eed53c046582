"""The row operators on hosts without a GPU."""

import os
import re
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
from zookeeper_amd import nn, ops
x = torch.randn(4, 40, requires_grad=True)
m = torch.nn.Sequential(nn.LayerNorm(40), nn.QuantDense(40, 8, use_bias=True, kept="int8"),
                        nn.GELU(kept="int8"))
r = ops.token_logprobs(m(x), torch.zeros(4, dtype=torch.int64), top=2)
(r.logp + r.entropy).sum().backward()
kept = ops.pack8(x.detach())
ops.dense8_grads(ops.unpack8(kept), kept)
assert x.grad.abs().sum() > 0
print("done")
"""


def test_a_torch_without_gpu_bindings(tmp_path):
    """A CPU build of torch has no ``torch._C._cuda_*``: the package imports, and the
    operators run on host tensors."""
    run = subprocess.run([sys.executable, "-c", PROGRAM], capture_output=True, text=True,
                         cwd=str(tmp_path), env=dict(os.environ, PYTHONPATH=ROOT), timeout=300)
    assert run.returncode == 0 and run.stdout.strip().endswith("done"), run.stderr[-2000:]


def test_no_shared_state_without_atomics():
    """The C entries are called from several host threads (the calls release the GIL): what
    they keep between calls is atomic or constant."""
    for name in ("act8.hip", "layer_norm.hip", "logprobs.hip", "rows.h"):
        with open(os.path.join(ROOT, "zookeeper_amd", "csrc", "kernels", name)) as f:
            for line in f:
                m = re.match(r"\s*static\s+(?!const|constexpr|__device__|std::atomic)(.*)", line)
                assert not m or re.match(r"[\w:<> *&]+\(", m.group(1)), (name, line)
