"""Log probabilities from hidden states: first calls, precision, large numbers of rows."""
import subprocess
import sys

import pytest

from mamba_tp_lite_b200 import build as B

pytestmark = pytest.mark.gpu

FIRST_CALL = """
import torch
from mamba_tp_lite_b200 import logprobs as P
dtype, top_k = torch.{dtype}, {top_k}
g = torch.Generator().manual_seed(0)
h = torch.randn(200, 64, generator=g).to(dtype).cuda()
w = torch.randn(1000, 64, generator=g).to(dtype).cuda()
t = torch.randint(0, 1000, (200,), generator=g).cuda()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = P.lm_head_logprobs(h, w, t, top_k=top_k)
graph.replay()
torch.cuda.synchronize()
want = P.lm_head_logprobs(h, w, t, top_k=top_k)
assert all(a is b or torch.equal(a, b) for a, b in zip(out, want))
"""


@pytest.mark.parametrize("dtype,top_k", [("bfloat16", 5), ("bfloat16", 0), ("float32", 5)])
def test_the_first_call_of_a_process_may_be_a_captured_one(dtype, top_k):
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.format(dtype=dtype, top_k=top_k)], cwd=B.REPO, timeout=300,
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
