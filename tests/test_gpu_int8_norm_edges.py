"""The norm with int8 output where its forms could part, and what lies around its results and around rows that are read back."""
import pytest
import torch

from mamba_tp_lite_b200 import _lib as L
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


# fp16 pairs (their bits) and an fp32 weight: the largest |y| of a row of such a pair and zeros is 127 t and one unit in the last
# place of a 64-bit number, t the middle between two fp32 numbers, where the product with 1 / 127 rounds otherwise than the quotient
BORDERS = {2: [("0x1.69880cp+6", -20296, -24234), ("0x1.697b8cp+6", -18826, 6391), ("0x1.69b676p+6", -19865, 6046),
               ("0x1.698af4p+6", 14871, -22293)],
           1024: [("0x1.ff75d2p+1", 17027, -20864), ("0x1.ff9404p+1", 15872, 8631), ("0x1.ffdd62p+1", 15897, -26133)],
           2048: [("0x1.69f292p+1", -16580, 11752)]}


@pytest.mark.parametrize("cols,weight,h0,h1", [(c, *b) for c in BORDERS for b in BORDERS[c]])
def test_a_scale_is_the_quotient_rounded_once(cols, weight, h0, h1):
    """max |y| / 127 in 64 bits, then to fp32, next to the middle between two fp32 numbers, in every form of the kernel.  The
    kernel's operations are followed one by one: the sum of two fp16 squares and its product with a power of two are exact."""
    w = torch.zeros(cols, device=dev())
    w[0] = float.fromhex(weight)
    x = torch.zeros(1, cols, device=dev(), dtype=F16)
    x[0, :2] = torch.tensor([h0, h1], dtype=torch.int16).view(F16).to(dev())
    d = x[0, :2].double()
    y = (d[0] * torch.rsqrt(d.square().sum() * (1.0 / cols) + float(torch.tensor(1e-5))) * w[0].double()).abs()
    by = torch.full_like(y, 127.0)
    want = (y / by).float()
    assert want != (y * (1.0 / by)).float()  # the row is one of those
    for rows in (1, 700):
        x, zero = x[:1].repeat(rows, 1), torch.zeros(rows, cols, device=dev())
        for q in [Q.rms_norm_int8(x, w, 1e-5), Q.rms_norm_int8(x.float(), w, 1e-5)] + [
                Q.add_rms_norm_int8(x.to(x_type), zero.to(r_type), w, 1e-5)[0]
                for x_type, r_type in [(F16, F16), (F16, F32), (F32, F32), (F32, F16)]]:
            assert (q.scale == want).all()


@pytest.mark.parametrize("cols", [40, 1024, 2051, 5120, 16400])
def test_scales_are_quotients_rounded_once(cols):
    """Rows of +-1 and eps 0: |y| is the weight.  (An fp32 number / 127 is never next to the middle between two others: the
    order of a sum does not matter.)"""
    g = gen(cols)
    x = (torch.rand(900, cols, generator=g, device=dev()) < 0.5) * 2.0 - 1
    w = torch.rand(cols, generator=g, device=dev()) + 0.5
    want = (w.double().amax() / torch.full((), 127.0, device=dev(), dtype=torch.float64)).float()
    for t in (F32, BF):
        assert (Q.rms_norm_int8(x.to(t), w, 0.0).scale == want).all()


@pytest.mark.parametrize("rows,cols", [(3, 96), (3, 101), (3, 4096), (700, 500), (700, 701), (700, 1111), (700, 2048), (3, 16400)])
@pytest.mark.parametrize("x_type,r_type", [(BF, F32), (F32, F32), (BF, BF), (F16, F16), (F32, BF), (BF, None), (F32, None)])
@pytest.mark.parametrize("left,right", [(0, 0), (16, 16), (3, 6)])
def test_what_lies_around_a_norm_s_outputs_stays(rows, cols, x_type, r_type, left, right):
    """Codes, scales and the stream inside wider and longer buffers, through the C entry point; also in place."""
    x = rows_of(rows, cols, x_type, cols, left, right)
    w = (1 + 0.3 * torch.randn(cols, generator=gen(3), device=dev()))
    wide = left + cols + right
    inside = (slice(2, 2 + rows), slice(left, left + cols))

    def guarded(dtype, value):
        return torch.full((rows + 4, wide), value, device=dev(), dtype=dtype)

    for inplace in ((False, True) if r_type else (False,)):
        codes, scale = guarded(torch.int8, 77), torch.full((rows + 4,), 7.0, device=dev())
        res_args, h, own = (None, 0, 0, None, 0), x, None
        if r_type:
            res = rows_of(rows, cols, r_type, cols + 1)
            own = guarded(r_type, 7.0)
            if inplace:
                own[inside] = res
                given = own[inside]
            else:
                given = res
            res_args = (given.data_ptr(), L.dtype_code(r_type), given.stride(0), own[inside].data_ptr(), wide)
            h = R.add(x, res)
        L.call("mtp_rmsnorm_int8", x.data_ptr(), L.dtype_code(x_type), x.stride(0), *res_args, rows, cols, w.data_ptr(), L.F32, 1e-5,
               codes[inside].data_ptr(), wide, scale[2:].data_ptr(), L.stream_ptr())
        R.check_rows(codes[inside], scale[2:2 + rows], R.norm(h, w, 1e-5))
        if own is not None:
            assert torch.equal(own[inside], h)
            own[inside] = 7.0
            assert (own == 7.0).all()
        codes[inside], scale[2:2 + rows] = 77, 7.0
        assert (codes == 77).all() and (scale == 7.0).all()


@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 8), (5, 13), (33, 100), (300, 1111), (40, 4096)])
@pytest.mark.parametrize("out", [F32, BF, F16])
@pytest.mark.parametrize("left,right", [(0, 8), (8, 8), (16, 0), (1, 0), (3, 6)])
def test_what_lies_around_rows_that_are_read_back_stays(rows, cols, out, left, right):
    """Results inside wider rows, on a vector's boundary and off it, through the C entry point."""
    codes = torch.randint(-127, 128, (rows, cols + 16), generator=gen(cols), device=dev()).to(torch.int8)
    scale = torch.rand(rows, generator=gen(rows), device=dev()) + 0.1
    held = torch.full((rows + 4, left + cols + right), 7.0, device=dev(), dtype=out)
    inside = held[2:2 + rows, left:left + cols]
    for at in (0, 8, 5):
        part = codes[:, at:at + cols]
        L.call("mtp_dequantize_rows", part.data_ptr(), cols + 16, scale.data_ptr(), rows, cols, inside.data_ptr(), L.dtype_code(out),
               held.stride(0), L.stream_ptr())
        assert torch.equal(inside, (part.float() * scale[:, None]).to(out))
        inside.fill_(7.0)
        assert (held == 7.0).all()


@pytest.mark.parametrize("b,l,d", [(2, 5, 96), (3, 70, 33)])
def test_in_place_beside_x_in_three_dimensions(b, l, d):
    buf = rows_of(b * l, 2 * d, BF, 7).reshape(b, l, 2 * d).clone()
    x, res = buf[:, :, :d], buf[:, :, d:]
    kept, want = x.clone(), R.add(x, res)
    w = 1 + 0.3 * torch.randn(d, generator=gen(3), device=dev())
    q, h = Q.add_rms_norm_int8(x, res, w, 1e-5, inplace=True)
    assert h is res and torch.equal(res, want) and torch.equal(x, kept)
    R.check_rows(q.codes.reshape(-1, d), q.scale.reshape(-1), R.norm(want, w, 1e-5).reshape(-1, d))
