"""Log probabilities from hidden states: first calls, precision, large numbers of rows."""
import subprocess
import sys

import numpy as np
import pytest
import torch

from mamba_tp_lite_b200 import build as B
from mamba_tp_lite_b200 import logprobs as P
from tests import logits_ref as R
from tests.gpu_util import dev
from tests.test_gpu_logprobs import BF, F32, check_score, close

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


def exact_inputs(rows, v, k, dtype):
    """R.exact_score_inputs on the GPU, its targets with one that is no token, and both with rows on 16-byte boundaries."""
    h, w = R.exact_score_inputs(rows, v, k, k)
    t = np.arange(rows) % v
    if rows > 1:
        t[1] = -1
    wide = (k + 7) // 8 * 8
    on = []
    for a in (h, w):
        buf = torch.full((len(a), wide), float("nan"), dtype=dtype, device=dev())
        buf[:, :k] = torch.from_numpy(a).to(dtype)
        on.append(buf[:, :k])
    return h, w, t, *on, torch.from_numpy(t).to(dev())


@pytest.mark.parametrize("rows,v,k", [(129, 255, 1024), (64, 50281, 768), (300, 2049, 2048), (1, 1001, 2048), (5, 777, 1100),
                                      (130, 1001, 2560), (70, 4001, 3000), (33, 333, 2120), (4200, 301, 1100)])
def test_scores_of_exact_sums(rows, v, k):
    """Logits without an error of their own but for one rounding where accumulators are joined: what is left is the
    softmax's.  One, two and three accumulators, of equal and unequal length; more rows than a group of tiles has."""
    h, w, t, hd, wd, td = exact_inputs(rows, v, k, BF)
    n = R.score_accumulators(k)
    _, lp, lp_bound, ent, ent_bound = R.exact_score_bounds(h, w, t, n if k > n else None)
    r = P.lm_head_logprobs(hd, wd, td)
    close(r.logprob, lp, lp_bound, "logprob")
    close(r.entropy, ent, ent_bound, "entropy")
    r = P.lm_head_logprobs(hd, wd, td, entropy=False)
    close(r.logprob, lp, lp_bound, "logprob without the entropy")


@pytest.mark.parametrize("rows,v,k", [(129, 255, 1024), (3, 5001, 1000), (300, 2049, 520)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_alternatives_of_exact_sums(rows, v, k, dtype):
    """The form that keeps logits, whose product sums K as a whole: the alternatives are those of the exact logits."""
    h, w, t, hd, wd, td = exact_inputs(rows, v, k, dtype)
    x, lp, lp_bound, ent, ent_bound = R.exact_score_bounds(h, w, t)
    r = P.lm_head_logprobs(hd, wd, td, top_k=20)
    close(r.logprob, lp, lp_bound, "logprob")
    close(r.entropy, ent, ent_bound, "entropy")
    ids = R.top(x, 20)
    np.testing.assert_array_equal(r.top_ids.cpu().numpy(), ids)
    want = np.take_along_axis(R.log_probs(x), ids, 1)
    close(r.top_logprobs, want, R.logprob_bound(x, want), "top_logprobs")
