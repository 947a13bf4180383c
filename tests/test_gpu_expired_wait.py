"""What scoring gives when a device wait of its pass has expired: NaN, never a value that could be taken for one.

The joining kernels are launched on partial statistics and status words made here (expired_wait.cu)."""
import ctypes as C
import subprocess

import numpy as np
import pytest
import torch

from mamba_tp_lite_b200 import _lib as L
from mamba_tp_lite_b200 import build as B
from mamba_tp_lite_b200 import logprobs as P
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu

LOWEST = torch.finfo(torch.float32).min


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    L.load()
    out = str(tmp_path_factory.mktemp("expired") / "expired_wait.so")
    src = f"{B.REPO}/tests/expired_wait.cu"
    subprocess.check_call([B.nvcc()] + B.ARCH + B.NVCC_FLAGS + ["-I", B.CSRC, "-shared", src, "-o", out, L.LIB_PATH,
                                                                "-Xlinker", "-rpath", "-Xlinker", B.PKG])
    return C.CDLL(out)


def join(kernels, m, s, u, hit, status, targets, vocab):
    """m, s, u [tiles][rows] as a pass leaves them; (logprob, entropy) of the rows at temperature 1."""
    tiles, rows = m.shape
    part = torch.stack([m, s, u]).to(dev())
    hit, status, targets = hit.to(dev()), status.to(dev()), targets.to(dev())
    lp, ent = torch.full((rows,), 7.0, device=dev()), torch.full((rows,), 7.0, device=dev())
    fn = kernels.test_score_join
    fn.argtypes = [C.c_void_p] * 4 + [C.c_int] * 4 + [C.c_void_p] * 3
    assert fn(L.ptr(targets), L.ptr(part), L.ptr(hit), L.ptr(status), len(status), rows, vocab, tiles, L.ptr(lp), L.ptr(ent),
              L.stream_ptr()) == 0
    torch.cuda.synchronize()
    return lp.cpu(), ent.cpu()


def passed(tiles, rows, seed=0):
    """Statistics of a pass over logits of which each tile holds two: x and x - 1."""
    g = torch.Generator().manual_seed(seed)
    m = torch.randn(tiles, rows, generator=g)
    e, y = np.exp(-1.0), -1.0 / np.log(2.0)
    return m, torch.full_like(m, 1 + e), torch.full_like(m, e * y)


@pytest.mark.parametrize("tiles,rows", [(1, 1), (1, 9), (3, 6), (300, 20)])
@pytest.mark.parametrize("lost", ["all", "some", "none"])
def test_scores_of_a_pass_whose_wait_expired_are_nan(kernels, tiles, rows, lost):
    """A CTA that gives up leaves (lowest, 0, 0) for its tiles and marks its status word.  Where all of a row's
    tiles are such, the joined row looks like one of -inf alone."""
    m, s, u = passed(tiles, rows)
    if lost != "none":
        gone = slice(None) if lost == "all" else slice(0, 1)
        m[gone], s[gone], u[gone] = LOWEST, 0.0, 0.0
    status = torch.zeros(148, dtype=torch.int32)
    status[147] = 1
    targets = torch.arange(rows) % 2  # tokens 0 and 1 of the first tile
    if rows > 2:
        targets[1], targets[2] = -1, 2 * tiles  # no token, and one past the vocabulary
    hit = torch.where(targets == 0, m[0], m[0] - 1)
    lp, ent = join(kernels, m, s, u, hit, status, targets, 2 * tiles)
    assert torch.isnan(ent).all()
    assert torch.isnan(lp[targets >= 0]).all()
    assert (lp[targets < 0] == 0).all()


def test_scores_of_a_pass_that_came_through(kernels):
    """The same statistics with no status word set: the definition, and a row of -inf alone among them."""
    tiles, rows = 5, 10
    m, s, u = passed(tiles, rows)
    m[:, 4], s[:, 4], u[:, 4] = LOWEST, 0.0, 0.0
    x = torch.stack([m, m - 1], 1).double().permute(2, 0, 1).reshape(rows, 2 * tiles)
    targets = torch.zeros(rows, dtype=torch.int64)
    hit = m[0].clone()
    hit[4] = float("-inf")
    lp, ent = join(kernels, m, s, u, hit, torch.zeros(3, dtype=torch.int32), targets, 2 * tiles)
    want = torch.log_softmax(x, -1)
    p = want.exp()
    ok = torch.arange(rows) != 4
    # ten terms of at most 2^-22 relative error each, a logarithm of at most 2^3: below 1e-5
    assert (lp[ok] - want[ok, 0]).abs().max() < 1e-5 and (ent[ok] + (p * want).sum(-1)[ok]).abs().max() < 1e-5
    assert lp[4] == float("-inf") and ent[4] == 0


@pytest.mark.parametrize("rows,v", [(1, 9), (1, 50280), (200, 3001), (2500, 200)])
@pytest.mark.parametrize("top_k", [0, 5])
def test_rows_of_a_product_whose_wait_expired_are_nan(kernels, rows, v, top_k):
    """Scoring in blocks: the product's logits are whatever the workspace held, so nothing that comes from them may look
    like a value.  With the word clear the results are those of the plain call."""
    x = (torch.randn(rows, v, generator=torch.Generator().manual_seed(rows)) * 3).to(dev())
    targets = (torch.arange(rows) % v).to(dev())
    if rows > 2:
        targets[1], targets[2] = -1, v
    want = P.token_logprobs(x, targets, top_k=top_k)
    fn = kernels.test_rows_after_a_product
    fn.argtypes = [C.c_void_p, C.c_int64, C.c_int] + [C.c_void_p] * 3 + [C.c_int] + [C.c_void_p] * 4
    for status in (0, 1):
        word = torch.tensor([status], dtype=torch.int32, device=dev())
        lp, ent = torch.full((rows,), 7.0, device=dev()), torch.full((rows,), 7.0, device=dev())
        ids = torch.zeros(rows, max(top_k, 1), dtype=torch.int64, device=dev())
        tlp = torch.full((rows, max(top_k, 1)), 7.0, device=dev())
        assert fn(L.ptr(x), rows, v, L.ptr(targets), L.ptr(lp), L.ptr(ent), top_k, L.ptr(ids), L.ptr(tlp), L.ptr(word),
                  L.stream_ptr()) == 0
        torch.cuda.synchronize()
        if status:
            assert torch.isnan(lp[targets >= 0]).all() and (lp[targets < 0] == 0).all() and torch.isnan(ent).all()
            assert top_k == 0 or (torch.isnan(tlp).all() and (ids >= 0).all() and (ids < v).all())
        else:
            for got, ref in ((lp, want.logprob), (ent, want.entropy)):
                assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(ref))
            assert top_k == 0 or (torch.equal(ids, want.top_ids) and torch.equal(tlp, want.top_logprobs))


@pytest.mark.parametrize("rows,dtype", [(300, torch.bfloat16), (16, torch.bfloat16), (300, torch.float32)])
def test_scoring_in_blocks_clears_its_status_word(rows, dtype):
    """The word lies in the workspace, which holds anything to start with: all ones here."""
    v, k, top_k = 700, 64, 3
    g = torch.Generator().manual_seed(rows)
    h = torch.randn(rows, k, generator=g).to(dtype).to(dev())
    w = torch.randn(v, k, generator=g).to(dtype).to(dev())
    args = (L.ptr(h), k, rows, k, L.ptr(w), k, v, L.dtype_code(dtype))
    need = C.c_int64(0)
    L.call("mtp_lm_head_logprobs_workspace", *args, top_k, C.byref(need))
    ws = torch.full((need.value,), 255, dtype=torch.uint8, device=dev())
    ent = torch.empty(rows, device=dev())
    ids, tlp = torch.empty(rows, top_k, dtype=torch.int64, device=dev()), torch.empty(rows, top_k, device=dev())
    L.call("mtp_lm_head_logprobs", *args, None, 1.0, None, L.ptr(ent), top_k, L.ptr(ids), L.ptr(tlp), L.ptr(ws), need.value,
           L.stream_ptr())
    want = P.lm_head_logprobs(h, w, top_k=top_k)
    assert torch.equal(ent, want.entropy) and torch.equal(tlp, want.top_logprobs) and torch.isfinite(ent).all()
