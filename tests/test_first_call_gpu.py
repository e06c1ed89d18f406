"""The first call of a process, made while a graph is captured: nothing that an operator sets up once may break the capture."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

HEAD = """
import torch
from rbruck_alltoallv_b200.ops.moe import linear_int8, moe_few_tokens, quantize_weight_int8
from rbruck_alltoallv_b200.ops.norm import block_norm
torch.manual_seed(0)
rand = lambda *n: torch.randn(*n, device="cuda").bfloat16()
x, logits, w13, w2 = rand(20, 64), torch.randn(20, 4, device="cuda"), rand(4, 80, 64), rand(4, 64, 40)
rows, (q, s) = rand(70, 64), quantize_weight_int8(rand(64, 64))
res, z, w = torch.randn(20, 64, device="cuda"), rand(20, 64), rand(64)
"""
CALLS = {
    "moe": "lambda: (moe_few_tokens(x[:1], logits[:1], w13, w2), moe_few_tokens(x, logits, w13, w2))",
    "int8": "lambda: (linear_int8(rows[:5], q, s), linear_int8(rows, q, s))",
    "norm": "lambda: block_norm(res, z, w, pre_weight=w)",
}
TAIL = """
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = call()
graph.replay()
want = call()
assert all(torch.equal(a, b) for a, b in zip(got, want)) and not any(a.isnan().any() for a in got)
"""


@pytest.mark.parametrize("name", CALLS)
def test_first_call_in_a_capture(name):
    done = subprocess.run([sys.executable, "-c", f"{HEAD}\ncall = {CALLS[name]}\n{TAIL}"], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
