"""What the int8 product gives when a device wait expires: NaN, never a value that could be taken for one; and it returns, with
nothing left behind that disturbs the next call."""
import ctypes as C
import subprocess

import pytest
import torch

from mamba_tp_lite_b200 import _lib as L
from mamba_tp_lite_b200 import build as B
from mamba_tp_lite_b200 import int8 as Q
from tests import int8_ref as R
from tests.gpu_util import dev
from tests.test_gpu_int8 import BF, codes_of

pytestmark = pytest.mark.gpu

SPLIT, TILE, PAIR = 0, 1, 2
# form, split, columns, (M, N, K): several tiles for a CTA, several rounds of the ring, rows and columns that end inside a tile
FORMS = [(SPLIT, 1, 64, (40, 300, 1000)), (SPLIT, 4, 64, (64, 256, 4096)), (SPLIT, 8, 128, (130, 1000, 8192)), (TILE, 1, 64, (256, 9000, 300)),
         (TILE, 1, 128, (1000, 4100, 2048)), (PAIR, 1, 256, (512, 12000, 300)), (PAIR, 1, 256, (1500, 5000, 2048))]


@pytest.fixture(scope="module")
def product(tmp_path_factory):
    L.load()
    so = str(tmp_path_factory.mktemp("int8") / "int8_expired_wait.so")
    subprocess.check_call([B.nvcc()] + B.ARCH + B.NVCC_FLAGS + ["-I", B.CSRC, "-shared", f"{B.REPO}/tests/int8_expired_wait.cu", "-o", so,
                                                                L.LIB_PATH, "-Xlinker", "-rpath", "-Xlinker", B.PKG])
    fn = C.CDLL(so).test_int8_linear
    fn.argtypes = [C.c_int] * 4 + [C.c_uint64, C.c_void_p, C.c_int64, C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_int64, C.c_void_p, C.c_int,
                   C.c_void_p, C.c_int64, C.c_void_p]

    def call(form, split, bn, lose, timeout_ns, a, w, pad):
        (m, k), n = a.codes.shape, w.codes.shape[0]
        held = torch.full((m + 2, n + pad), 7.0, device=dev(), dtype=BF)
        assert fn(form, split, bn, lose, timeout_ns, L.ptr(a.codes), a.codes.stride(0), L.ptr(a.scale), m, k, L.ptr(w.codes),
                  w.codes.stride(0), L.ptr(w.scale), n, L.ptr(held), n + pad, L.stream_ptr()) == 0
        torch.cuda.synchronize()
        assert (held[m:] == 7).all() and (held[:, n:] == 7).all()
        return held[:m, :n]

    return call


@pytest.mark.parametrize("pad", [8, 5])  # results by TMA or 16-byte stores, and one by one
@pytest.mark.parametrize("form,split,bn,size", FORMS)
def test_results_of_an_expired_wait_are_nan(product, form, split, bn, size, pad):
    m, n, k = size
    pad += -n % 8
    a, w = codes_of(m, k, 1, -k % 16), codes_of(n, k, 2, -k % 16)
    want = R.linear(a.codes, a.scale, w.codes, w.scale, None, BF)
    assert torch.equal(product(form, split, bn, 0, 2000000000, a, w, pad), want)  # the same call with all its bytes
    for _ in range(2):
        assert torch.isnan(product(form, split, bn, 1, 5000000, a, w, pad)).all()
        assert torch.equal(product(form, split, bn, 0, 2000000000, a, w, pad), want)
    assert torch.equal(Q.int8_linear(a, w), want)
