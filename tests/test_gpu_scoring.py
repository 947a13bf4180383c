"""Log probabilities from hidden states: first calls, precision, large numbers of rows."""
import subprocess
import sys

import pytest
import torch

from mamba_tp_lite_b200 import build as B
from mamba_tp_lite_b200 import logprobs as P
from tests.gpu_util import dev
from tests.test_gpu_logprobs import BF, F32, check_score

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


@pytest.mark.parametrize("dtype,v,k", [(F32, 3, 8), (F32, 1, 1), (BF, 5, 3)])
def test_more_rows_than_a_product_takes_at_once(dtype, v, k):
    """4.2 million rows through the form that keeps logits, whose CUDA-core product has 65535 x 64 places for rows."""
    rows = 65536 * 64 + 77
    g = torch.Generator(device=dev()).manual_seed(v)
    h = torch.randn(rows, k, generator=g, device=dev()).to(dtype)
    w = torch.randn(v, k, generator=g, device=dev()).to(dtype)
    t = torch.randint(0, v, (rows,), generator=g, device=dev())
    r = P.lm_head_logprobs(h, w, t, top_k=1)
    edge = 65535 // 2 * 128
    for part in (slice(0, 50), slice(edge - 50, edge + 50), slice(rows - 50, rows)):
        check_score(h[part], w, t[part], P.TokenLogprobs(r.logprob[part], r.entropy[part], None, None))
    assert torch.isfinite(r.logprob).all() and (r.top_ids < v).all() and (r.top_ids >= 0).all()
