"""The norm with int8 output where its forms could part."""
import pytest
import torch

from mamba_tp_lite_b200 import int8 as Q
from tests import int8_ref as R
from tests.gpu_util import dev
from tests.test_gpu_int8 import BF, F16, F32, gen, rows_of

pytestmark = pytest.mark.gpu


# 3 rows: 8 values a thread; 700: by warps to 768 columns, then by CTAs with 16, 24 or 32 values a thread
@pytest.mark.parametrize("rows,cols", [(3, 24), (3, 1111), (3, 2048), (3, 9000), (700, 500), (700, 701), (700, 1111), (700, 1536),
                                       (700, 2048)])
@pytest.mark.parametrize("x_type", [BF, F16])
@pytest.mark.parametrize("residual", ["none", "same", "f32"])
def test_a_weight_at_every_offset(rows, cols, x_type, residual):
    """Weights side by side in one buffer: every offset within 32 bytes, in each type, gives what a weight of its own gives."""
    x = rows_of(rows, cols, x_type, cols)
    res = None if residual == "none" else rows_of(rows, cols, x_type if residual == "same" else F32, cols + 1)
    h = x if res is None else R.add(x, res)

    def call(w):
        return Q.rms_norm_int8(x, w, 1e-5) if res is None else Q.add_rms_norm_int8(x, res, w, 1e-5)[0]

    for w_type in (F32, BF, F16):
        flat = (1 + 0.3 * torch.randn(cols + 16, generator=gen(3), device=dev())).to(w_type)
        for at in range(32 // flat.element_size()):
            w = flat[at:at + cols]
            q = call(w)
            R.check_rows(q.codes, q.scale, R.norm(h, w, 1e-5))
            own = call(w.clone())
            assert torch.equal(q.codes, own.codes) and torch.equal(q.scale, own.scale)
