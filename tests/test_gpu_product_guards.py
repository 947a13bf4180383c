"""What lies beside and behind a matrix product's results in a wider buffer stays as it was, wherever a row of them ends."""
import pytest
import torch

from mamba_tp_lite_b200 import _lib as L
from tests import int8_ref as R
from tests.gpu_util import dev
from tests.test_gpu_int8 import F32, TYPES, codes_of

pytestmark = pytest.mark.gpu


def guarded(m, n, pad, dtype):
    """A buffer of sevens with rows a multiple of 16 bytes apart where pad is 0, and its first m rows of n columns."""
    wide = n + (-n % 8) + 8 + pad
    held = torch.full((m + 3, wide), 7.0, device=dev(), dtype=dtype)
    return held, held[:m, :n]


# up to 16 rows, K over a cluster, tiles of 64 and 128 columns, pairs of CTAs
@pytest.mark.parametrize("m,k", [(3, 64), (16, 4096), (40, 512), (130, 2048), (256, 64), (700, 256), (2100, 128)])
@pytest.mark.parametrize("n", [1, 3, 100, 257, 700, 1031, 4099, 4100, 4102])
@pytest.mark.parametrize("pad", [0, 1])
def test_int8_product(m, k, n, pad):
    a, w = codes_of(m, k, 1), codes_of(n, k, 2)
    bias = torch.arange(n, device=dev(), dtype=F32)
    for t in TYPES:
        held, out = guarded(m, n, pad, t)
        L.call("mtp_int8_linear", a.codes.data_ptr(), k, a.scale.data_ptr(), m, k, w.codes.data_ptr(), k, w.scale.data_ptr(), n,
               bias.data_ptr(), L.F32, out.data_ptr(), L.dtype_code(t), held.stride(0), L.stream_ptr())
        assert torch.equal(out, R.linear(a.codes, a.scale, w.codes, w.scale, bias, t))
        out.fill_(7.0)
        assert (held == 7.0).all()


@pytest.mark.parametrize("m,k", [(3, 64), (20, 64), (33, 512), (130, 2048), (700, 256)])
@pytest.mark.parametrize("n", [1, 16, 100, 257, 700, 1031, 4099, 4100, 4102])
@pytest.mark.parametrize("pad", [0, 1])
def test_bf16_product(m, k, n, pad):
    """Whole numbers: the sums are exact in fp32, in any order."""
    g = torch.Generator(device=dev()).manual_seed(k)
    a, w = (torch.randint(-4, 5, (r, k), generator=g, device=dev()).to(torch.bfloat16) for r in (m, n))
    bias = (torch.arange(n, device=dev()) % 7).to(F32)
    want = a.double() @ w.double().T
    for t in (F32, torch.bfloat16):
        for epi, b in ((L.EPI_STORE, None), (L.EPI_BIAS, bias)):
            held, out = guarded(m, n, pad, t)
            L.call("mtp_gemm", L.ptr(a), L.ptr(w), L.ptr(out), m, n, k, k, k, held.stride(0), L.BF16, L.dtype_code(t), epi, L.ptr(b),
                   L.F32, L.stream_ptr())
            assert torch.equal(out, (want if b is None else want + b.double()).to(t))
            out.fill_(7.0)
            assert (held == 7.0).all()
