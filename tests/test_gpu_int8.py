"""The 8-bit linear path on the GPU against its definitions in 64 bits (int8_ref.py has the bounds)."""
import subprocess
import sys

import pytest
import torch

from mamba_tp_lite_b200 import build as B
from mamba_tp_lite_b200 import int8 as Q
from tests import int8_ref as R
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu

F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF, F16]


def gen(seed):
    return torch.Generator(device=dev()).manual_seed(seed)


def rows_of(rows, cols, dtype, seed, pad=0, offset=0, scale=1.0):
    """Rows of normal values, some tokens and channels louder, cut out of wider rows at an offset."""
    g = gen(seed)
    x = torch.randn(rows, cols + pad + offset, generator=g, device=dev()) * scale
    x *= torch.exp(torch.randn(rows, 1, generator=g, device=dev()))
    return x.to(dtype)[:, offset:offset + cols]


def codes_of(rows, cols, seed, pad=0, offset=0, extreme=False):
    g = gen(seed)
    c = torch.randint(-128, 128, (rows, cols + pad + offset), generator=g, device=dev(), dtype=torch.int64).to(torch.int8)
    if extreme:
        c.fill_(-128)
    return Q.Int8Rows(c[:, offset:offset + cols], torch.rand(rows, generator=g, device=dev()) * 0.1 + 1e-3)


# ------------------------------------------------------------------ rows
SHAPES = [(1, 1), (1, 2), (3, 7), (2, 15), (5, 16), (1, 17), (4, 31), (9, 64), (2, 255), (3, 256), (7, 1000), (1, 2048), (33, 2048),
          (5, 2051), (2, 4096), (1, 4097), (3, 5120), (2, 8192), (2, 8200), (2, 20000), (1, 131071), (1300, 96), (40000, 8)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize(rows, cols, dtype):
    x = rows_of(rows, cols, dtype, rows + cols)
    r = Q.quantize_rows(x)
    assert r.codes.shape == x.shape and r.scale.shape == (rows,)
    R.check_rows(r.codes, r.scale, x)
    for out in TYPES:
        want = (r.codes.float() * r.scale.unsqueeze(-1)).to(out)
        assert torch.equal(Q.dequantize_rows(r, out), want)


@pytest.mark.parametrize("pad,offset", [(0, 1), (1, 0), (3, 5), (8, 0), (16, 8), (8, 4)])
@pytest.mark.parametrize("cols", [1, 33, 512, 1111, 9000])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_of_strided_rows(pad, offset, cols, dtype):
    x = rows_of(6, cols, dtype, cols, pad, offset)
    r = Q.quantize_rows(x)
    R.check_rows(r.codes, r.scale, x)
    s = Q.quantize_rows(x.contiguous())
    assert torch.equal(r.codes, s.codes) and torch.equal(r.scale, s.scale)
    wide = torch.full((6, cols + pad + 9), 99, device=dev(), dtype=torch.int8)
    wide[:, offset:offset + cols] = r.codes
    got = Q.dequantize_rows(Q.Int8Rows(wide[:, offset:offset + cols], r.scale), dtype)
    assert torch.equal(got, (r.codes.float() * r.scale.unsqueeze(-1)).to(dtype))


@pytest.mark.parametrize("cols", [3, 8, 1000, 4096, 30000])
def test_quantize_of_rows_of_every_kind(cols):
    """Zeros, a NaN, infinities, values below the scale's floor, subnormals, the largest, ties between two codes."""
    top = torch.finfo(F32).max
    x = rows_of(12, cols, F32, cols).contiguous()
    x[0] = 0
    x[1, cols // 2] = float("nan")
    x[2, cols - 1] = float("inf")
    x[3, 0] = float("-inf")
    x[4] *= 1e-12
    x[5] = 1e-40
    x[6, 0], x[6, 1] = top, -top
    x[7, 0], x[7, 1:] = 127.0, (torch.arange(cols - 1, device=dev()) % 127) + 0.5  # scale 1: every code is a tie
    x[8, 0], x[8, 1:] = -254.0, -((torch.arange(cols - 1, device=dev()) % 127) * 2 + 1.0)  # the same with scale 2
    x[9, -1] = 1e30
    r = Q.quantize_rows(x)
    R.check_rows(r.codes, r.scale, x)
    assert torch.equal(r.codes[7, 1:].double(), torch.round(x[7, 1:].double()))
    assert torch.equal(r.codes[8, 1:].double(), torch.round(x[8, 1:].double() / 2))
    assert torch.isnan(Q.dequantize_rows(r)[1:4]).all()


@pytest.mark.parametrize("dtype", [BF, F16])
def test_codes_next_to_a_border(dtype):
    """Every value of a 16-bit type below the largest of its row: quotients as near to a half as the type has them."""
    bits = torch.arange(0, 0x7f80 if dtype == BF else 0x7c00, device=dev(), dtype=torch.int32).to(torch.int16).view(dtype)
    tops = [1.0, 3.3, 100.7, 254.0, 60000.0]
    x = torch.stack([torch.where(bits.float() < t, bits, torch.zeros_like(bits)) for t in tops])
    x[:, 0] = torch.tensor(tops, device=dev()).to(dtype)
    r = Q.quantize_rows(x)
    R.check_rows(r.codes, r.scale, x)
    want = torch.round(x.double() / r.scale.double().unsqueeze(-1))  # the quotient's rounding cannot reach a half: see int8_ref
    assert torch.equal(r.codes.double(), want)


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("x_type,r_type", [(F32, F32), (BF, F32), (BF, BF), (F16, F32), (F16, F16), (F32, BF), (BF, F16)])
def test_add_norm(rows, cols, x_type, r_type):
    x = rows_of(rows, cols, x_type, rows + cols, scale=0.3)
    res = rows_of(rows, cols, r_type, rows + cols + 1)
    w = 1 + 0.3 * torch.randn(cols, generator=gen(3), device=dev())
    for weight in (w, w.to(x_type)):
        q, h = Q.add_rms_norm_int8(x, res, weight, 1e-5)
        assert torch.equal(h, R.add(x, res))
        R.check_rows(q.codes, q.scale, R.norm(h, weight, 1e-5))
    own = res.clone()
    q2, h2 = Q.add_rms_norm_int8(x, own, weight, 1e-5, inplace=True)
    assert h2.data_ptr() == own.data_ptr() and torch.equal(own, h)
    assert torch.equal(q2.codes, q.codes) and torch.equal(q2.scale, q.scale)


@pytest.mark.parametrize("cols", [500, 701, 768, 769, 1000, 1024, 1025, 1200, 1335, 1536, 1537, 2048, 5120])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_many_rows(cols, dtype):
    x = rows_of(700, cols, dtype, cols)
    x[0::5] *= x[0::5].abs().amax(-1, keepdim=True).reciprocal() * 127  # steps of 1: ties
    x[0::5] = (x[0::5] * 2).round() / 2
    q = Q.quantize_rows(x)
    R.check_rows(q.codes, q.scale, x)
    assert torch.equal(q.codes[0::5].double(), (x[0::5].double() / q.scale[0::5].double().unsqueeze(-1)).round().clamp(-127, 127))


# many rows: codes next to a border, and rows whose largest product stands in several places
@pytest.mark.parametrize("cols", [500, 701, 768, 1000, 1001, 1200, 1536, 2048, 2051, 5120])
@pytest.mark.parametrize("x_type,r_type", [(F32, F32), (BF, F32), (BF, BF), (F16, F32), (F16, F16), (F32, None), (BF, None), (F16, None)])
def test_norm_of_many_rows(cols, x_type, r_type):
    x = rows_of(700, cols, x_type, cols)
    x[:, 7::97] = x[:, 7:8]
    w = 1 + 0.3 * torch.randn(cols, generator=gen(3), device=dev())
    w[7::97] = 40.0
    for weight in (w, w.to(BF)):
        if r_type is None:
            q, h = Q.rms_norm_int8(x, weight, 1e-5), x
        else:
            res = rows_of(700, cols, r_type, cols + 1)
            res[:, 7::97] = res[:, 7:8]
            q, h = Q.add_rms_norm_int8(x, res, weight, 1e-5)
            assert torch.equal(h, R.add(x, res))
        R.check_rows(q.codes, q.scale, R.norm(h, weight, 1e-5))


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_without_a_residual(rows, cols, dtype):
    x = rows_of(rows, cols, dtype, rows + cols)
    w = (1 + 0.3 * torch.randn(cols, generator=gen(3), device=dev())).to(dtype)
    q = Q.rms_norm_int8(x, w, 1e-5)
    R.check_rows(q.codes, q.scale, R.norm(x, w, 1e-5))


@pytest.mark.parametrize("pad,offset", [(0, 1), (3, 5), (8, 0), (16, 8)])
@pytest.mark.parametrize("cols", [1, 33, 512, 1111, 9000])
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_strided_rows(pad, offset, cols, dtype):
    x, res = rows_of(5, cols, dtype, cols, pad, offset), rows_of(5, cols, F32, cols + 1, offset, pad)
    w = rows_of(1, cols, dtype, 9, 1, 1)[0]
    q, h = Q.add_rms_norm_int8(x, res, w, 1e-6)
    assert torch.equal(h, R.add(x, res))
    R.check_rows(q.codes, q.scale, R.norm(h, w, 1e-6))
    held = rows_of(5, cols, F32, cols + 1, offset, pad + 2)
    own = held[:, :cols]  # in place, inside wider rows that stay as they are
    around = held._base[:, :pad].clone() if held._base is not None and pad else None
    want = R.add(x, own)
    Q.add_rms_norm_int8(x, own, w, 1e-6, inplace=True)
    assert torch.equal(own, want)
    if around is not None:
        assert torch.equal(held._base[:, :pad], around)


@pytest.mark.parametrize("cols", [3, 8, 1000, 4096, 30000])
def test_norm_of_rows_of_every_kind(cols):
    x = rows_of(10, cols, F32, cols).contiguous()
    x[0] = 0
    x[1, cols // 2] = float("nan")
    x[2, cols - 1] = float("inf")
    x[3] *= 1e-25   # squares below fp32's range
    x[4] *= 1e25    # squares above it
    x[5] = 1e-40
    x[6, 0], x[6, 1:] = 3e38, 0
    w = 1 + 0.3 * torch.randn(cols, generator=gen(3), device=dev())
    for eps in (1e-5, 0.0):
        q = Q.rms_norm_int8(x, w, eps)
        R.check_rows(q.codes, q.scale, R.norm(x, w, eps))  # eps 0: a row of zeros is 0 / 0
    w[1] = float("nan")
    assert torch.isnan(Q.rms_norm_int8(x, w, 1e-5).scale).all()
    w[1] = 1e38
    q = Q.rms_norm_int8(x[7:], w, 1e-5)
    R.check_rows(q.codes, q.scale, R.norm(x[7:], w, 1e-5))


def test_sums_that_overflow_a_16_bit_stream():
    x = torch.full((3, 100), 60000.0, device=dev(), dtype=F16)
    res = torch.full((3, 100), 60000.0, device=dev(), dtype=F16)
    res[1] = -60000.0
    q, h = Q.add_rms_norm_int8(x, res, torch.ones(100, device=dev()), 1e-5)
    assert torch.isinf(h[0]).all() and (h[1] == 0).all()
    assert torch.isnan(q.scale[0]) and (q.codes[0] == 0).all() and not torch.isnan(q.scale[1])


def test_leading_dimensions():
    x = rows_of(2 * 3 * 5, 96, BF, 0).view(2, 3, 5, 96)
    cut = x[:, :, 1:]
    r = Q.quantize_rows(cut)
    assert r.codes.shape == cut.shape and r.scale.shape == cut.shape[:-1]
    R.check_rows(r.codes.reshape(-1, 96), r.scale.reshape(-1), cut.reshape(-1, 96))
    t = x[0].transpose(0, 2)  # rows that are not dense
    r = Q.quantize_rows(t)
    R.check_rows(r.codes.reshape(-1, 3), r.scale.reshape(-1), t.reshape(-1, 3))
    one = Q.quantize_rows(x[0, 0, 0])
    assert one.codes.shape == (96,) and one.scale.shape == ()
    w = Q.quantize_rows(torch.randn(40, 96, generator=gen(1), device=dev()))
    assert Q.int8_linear(one, w).shape == (40,)
    r = Q.quantize_rows(cut)
    y = Q.int8_linear(r, w, dtype=F32)
    assert y.shape == (2, 3, 4, 40)
    assert torch.equal(y[1, 2], Q.int8_linear(Q.Int8Rows(r.codes[1, 2], r.scale[1, 2]), w, dtype=F32))
    same = x[0, 0, :1].expand(4, 96)  # one row four times
    r = Q.quantize_rows(same)
    R.check_rows(r.codes, r.scale, same)
    q, h = Q.add_rms_norm_int8(same, same, torch.ones(96, device=dev()), 1e-5)
    assert torch.equal(h, R.add(same, same)) and (q.codes == q.codes[0]).all()


def test_nothing_to_do():
    e = torch.empty(0, 40, device=dev(), dtype=BF)
    r = Q.quantize_rows(e)
    assert r.codes.shape == (0, 40) and r.scale.shape == (0,)
    assert Q.dequantize_rows(r).shape == (0, 40)
    q, h = Q.add_rms_norm_int8(e, e.float(), torch.ones(40, device=dev()))
    assert q.codes.shape == (0, 40) and h.shape == (0, 40)
    w = codes_of(7, 40, 0)
    assert Q.int8_linear(r, w).shape == (0, 7)
    assert Q.int8_linear(w, r).shape == (7, 0)
    assert Q.int8_linear(Q.Int8Rows(r.codes.view(3, 0, 40), r.scale.view(3, 0)), w).shape == (3, 0, 7)


# ------------------------------------------------------------------ products
def check_linear(a, w, bias=None, types=TYPES):
    for t in types:
        got = Q.int8_linear(a, w, bias, dtype=t)
        assert got.dtype == t
        want = R.linear(a.codes, a.scale, w.codes, w.scale, bias, t)
        assert torch.equal(got, want), f"{t}: {(got.float() - want.float()).abs().max().item()}"


SIZES = [(1, 1, 1), (1, 5, 3), (1, 16, 16), (1, 777, 1001), (1, 2048, 4096), (1, 8192, 2048), (2, 64, 64), (3, 100, 48), (4, 333, 128),
         (5, 256, 2048), (8, 1000, 512), (8, 2048, 4096), (9, 130, 96), (15, 64, 80), (16, 4096, 1024), (16, 129, 5120), (17, 128, 128),
         (31, 300, 272), (32, 2048, 4096), (33, 8192, 2048), (48, 65, 1040), (64, 2048, 4096), (65, 160, 144), (96, 1024, 512),
         (127, 256, 256), (128, 256, 128), (129, 257, 144), (200, 1000, 1000), (256, 512, 2048), (300, 777, 1008), (333, 777, 1001),
         (513, 2048, 768), (1000, 100, 64), (1025, 640, 16), (2048, 2304, 2560), (4099, 24, 32), (3, 50280, 64),
         (2500, 4100, 1000), (4099, 3001, 300), (5000, 6400, 128), (20, 10240, 2560), (100, 10240, 2560), (70, 50280, 64), (16, 20000, 2064),
         (130, 2048, 4096), (255, 1001, 2064), (256, 200, 8192), (192, 70, 20000), (250, 1024, 2048), (256, 2048, 4112)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(m, n, k):
    a, w = codes_of(m, k, 1), codes_of(n, k, 2)
    check_linear(a, w)
    bias = torch.randn(n, generator=gen(3), device=dev())
    check_linear(a, w, bias)
    check_linear(a, w, bias.to(BF), [BF])
    check_linear(a, w, bias.to(F16), [F16])


@pytest.mark.parametrize("m", [1, 2, 8, 16, 17, 40, 64, 128, 130, 700])
@pytest.mark.parametrize("pad,offset", [(0, 1), (3, 4), (5, 0), (16, 0), (16, 16), (24, 8)])
def test_linear_of_strided_rows(m, pad, offset):
    for n, k in [(70, 33), (200, 512), (256, 1000)]:
        check_linear(codes_of(m, k, 1, pad, offset), codes_of(n, k, 2), None, [BF, F32])
        check_linear(codes_of(m, k, 1), codes_of(n, k, 2, pad, offset), None, [BF, F32])


@pytest.mark.parametrize("m", [1, 5, 16, 17, 40, 128, 129, 700, 2600])
@pytest.mark.parametrize("n,k", [(70, 1), (130, 15), (64, 17), (100, 100), (1030, 257), (300, 1001), (2100, 2049)])
def test_what_lies_behind_a_row_is_not_summed(m, n, k):
    """Rows on 16-byte boundaries, with other codes between them."""
    pad = -k % 16 or 16
    check_linear(codes_of(m, k, 1, pad), codes_of(n, k, 2, pad), None, [F32])


@pytest.mark.parametrize("m", [1, 3, 16, 40, 128, 300])
def test_the_largest_sums(m):
    """-128 * -128 over 131071 columns is 2147467264, below 2^31."""
    a, w = codes_of(m, 131071, 1, extreme=True), codes_of(70, 131071, 2, extreme=True)
    check_linear(a, w, None, [F32])
    held = torch.zeros(m, 131072, device=dev(), dtype=torch.int8)  # the same on 16-byte boundaries
    held[:, :131071] = -128
    wide = torch.full((70, 131072), 77, device=dev(), dtype=torch.int8)  # what lies behind a row is not read into a sum
    wide[:, :131071] = -128
    check_linear(Q.Int8Rows(held[:, :131071], a.scale), Q.Int8Rows(wide[:, :131071], w.scale), None, [F32])
    wide[:, :131071] = 127
    check_linear(Q.Int8Rows(held[:, :131071], a.scale), Q.Int8Rows(wide[:, :131071], w.scale), None, [F32])


@pytest.mark.parametrize("m", [1, 9, 64, 300])
def test_scales_and_biases_that_are_not_finite(m):
    a, w = codes_of(m, 64, 1), codes_of(100, 64, 2)
    bias = torch.zeros(100, device=dev())
    a.scale[m - 1], w.scale[7], bias[9], w.scale[11] = float("nan"), float("nan"), float("inf"), 0.0
    a.codes[m - 1] = 0
    got = Q.int8_linear(a, w, bias, dtype=F32)
    want = R.linear(a.codes, a.scale, w.codes, w.scale, bias, F32)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.isnan(got[m - 1]).all() and torch.isnan(got[:, 7]).all()
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.parametrize("n", [64, 100, 2048])
def test_a_row_depends_on_no_other(n):
    a, w = codes_of(400, 512, 1), codes_of(n, 512, 2)
    full = Q.int8_linear(a, w, dtype=F32)
    for m in (1, 2, 7, 16, 17, 64, 100, 128, 129, 256):
        assert torch.equal(Q.int8_linear(Q.Int8Rows(a.codes[:m], a.scale[:m]), w, dtype=F32), full[:m])


def test_rows_behind_the_last_stay_as_they_were():
    """Outputs inside wider buffers, through the C entry points."""
    from mamba_tp_lite_b200 import _lib as L

    for m, n, k in [(5, 100, 64), (40, 96, 64), (130, 200, 64), (300, 264, 128)]:
        a, w = codes_of(m, k, 1), codes_of(n, k, 2)
        for t in TYPES:
            held = torch.full((m + 3, n + 8), 7.0, device=dev(), dtype=t)
            L.call("mtp_int8_linear", a.codes.data_ptr(), k, a.scale.data_ptr(), m, k, w.codes.data_ptr(), k, w.scale.data_ptr(), n,
                   None, 0, held.data_ptr(), L.dtype_code(t), n + 8, L.stream_ptr())
            assert torch.equal(held[:m, :n], R.linear(a.codes, a.scale, w.codes, w.scale, None, t))
            assert (held[m:] == 7).all() and (held[:, n:] == 7).all()
    x = rows_of(5, 100, BF, 0)
    codes = torch.full((7, 160), 77, device=dev(), dtype=torch.int8)
    scale = torch.full((7,), 7.0, device=dev())
    L.call("mtp_quantize_rows", x.data_ptr(), L.BF16, 100, 5, 100, codes.data_ptr(), 160, scale.data_ptr(), L.stream_ptr())
    R.check_rows(codes[:5, :100], scale[:5], x)
    assert (codes[5:] == 77).all() and (codes[:, 100:] == 77).all() and (scale[5:] == 7).all()


def test_offsets_past_32_bits():
    """A result of more than 2^31 values, rows of more than 2^31 values in all."""
    m, n, k = 70001, 40008, 16
    a, w = codes_of(m, k, 1), codes_of(n, k, 2)
    y = Q.int8_linear(a, w, dtype=BF)
    for part in (slice(0, 3), slice(53680, 53690), slice(m - 5, m)):
        assert torch.equal(y[part], R.linear(a.codes[part], a.scale[part], w.codes, w.scale, None, BF))
    q = Q.quantize_rows(y)
    for part in (slice(0, 3), slice(53680, 53690), slice(m - 5, m)):
        R.check_rows(q.codes[part], q.scale[part], y[part])
    back = Q.dequantize_rows(q, BF)
    for part in (slice(0, 3), slice(53680, 53690), slice(m - 5, m)):
        assert torch.equal(back[part], (q.codes[part].float() * q.scale[part].unsqueeze(-1)).to(BF))
    del back
    weight = torch.ones(n, device=dev(), dtype=BF)
    q, h = Q.add_rms_norm_int8(y, y, weight, 1e-5)
    for part in (slice(0, 3), slice(53680, 53690), slice(m - 5, m)):
        assert torch.equal(h[part], R.add(y[part], y[part]))
        R.check_rows(q.codes[part], q.scale[part], R.norm(h[part], weight, 1e-5))


def test_millions_of_short_rows():
    rows, k, n = 3_000_001, 16, 24
    x = rows_of(rows, k, BF, 5)
    q, h = Q.add_rms_norm_int8(x, x, torch.ones(k, device=dev()), 1e-5)
    R.check_rows(q.codes, q.scale, R.norm(h, torch.ones(k, device=dev()), 1e-5))
    r = Q.quantize_rows(x)
    R.check_rows(r.codes, r.scale, x)
    assert torch.equal(Q.dequantize_rows(r, BF), (r.codes.float() * r.scale.unsqueeze(-1)).to(BF))
    w = codes_of(n, k, 2)
    assert torch.equal(Q.int8_linear(r, w, dtype=F32), R.linear(r.codes, r.scale, w.codes, w.scale, None, F32))
    odd = Q.Int8Rows(r.codes[:, :13], r.scale)  # off 16-byte boundaries
    w = codes_of(n, 13, 2)
    assert torch.equal(Q.int8_linear(odd, w, dtype=BF), R.linear(odd.codes, odd.scale, w.codes, w.scale, None, BF))


# ------------------------------------------------------------------ as they are used
def boundary(x, res, out_w, norm_w, in_w):
    """From a layer's scan output to the next layer's in_proj output."""
    branch = Q.int8_linear(Q.quantize_rows(x), out_w, dtype=F32)
    rows, h = Q.add_rms_norm_int8(branch, res, norm_w, 1e-5)
    return Q.int8_linear(rows, in_w, dtype=BF), h


def boundary_inputs(rows, seed, d=256, e=512):
    x, res = rows_of(rows, e, BF, seed), rows_of(rows, d, F32, seed + 1)
    norm_w = rows_of(1, d, BF, seed + 2)[0]
    out_w = Q.quantize_rows(torch.randn(d, e, generator=gen(seed + 3), device=dev()) / 16)
    in_w = Q.quantize_rows(torch.randn(2 * e, d, generator=gen(seed + 4), device=dev()) / 16)
    return x, res, out_w, norm_w, in_w


@pytest.mark.parametrize("rows", [1, 4, 33, 200])
def test_a_run_of_them(rows):
    """Against the same definitions one after the other; the first quantiser's error bounds the first product:
    |error| <= scale / 2 per value."""
    x, res, out_w, norm_w, in_w = boundary_inputs(rows, 10)
    y, h = boundary(x, res, out_w, norm_w, in_w)
    q = Q.quantize_rows(x)
    R.check_rows(q.codes, q.scale, x)
    branch = R.linear(q.codes, q.scale, out_w.codes, out_w.scale, None, F32)
    assert torch.equal(h, R.add(branch, res))
    exact = x.double() @ (out_w.codes.double() * out_w.scale.double().unsqueeze(-1)).T
    step = (q.scale.double() / 2).unsqueeze(-1) * (out_w.codes.double().abs().sum(1) * out_w.scale.double())
    assert ((branch.double() - exact).abs() <= step * (1 + 1e-5) + 1e-6 * exact.abs()).all()
    q, _ = Q.add_rms_norm_int8(branch, res, norm_w, 1e-5)
    R.check_rows(q.codes, q.scale, R.norm(h, norm_w, 1e-5))
    assert torch.equal(y, R.linear(q.codes, q.scale, in_w.codes, in_w.scale, None, BF))


@pytest.mark.parametrize("rows", [1, 20, 200])
def test_captured_and_replayed(rows):
    """Two graphs and eager calls between their replays, on new inputs; a first call that is captured."""
    sets = [list(boundary_inputs(rows, s)) for s in (20, 40)]
    graphs, outs = [], []
    for s in sets:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(boundary(*s))
        graphs.append(g)
    for turn in range(3):
        for s in sets:
            s[0].copy_(rows_of(rows, 512, BF, 100 + turn))
        graphs[0].replay()
        other = boundary(*sets[1])
        graphs[1].replay()
        for s, out in zip(sets, outs):
            for got, want in zip(out, boundary(*s)):
                assert torch.equal(got, want)
        assert torch.equal(other[0], outs[1][0])


FIRST_CALL = """
import torch
from mamba_tp_lite_b200 import int8 as Q
g = torch.Generator().manual_seed(0)
x = torch.randn({rows}, 512, generator=g).to(torch.bfloat16).cuda()
r = torch.randn({rows}, 512, generator=g).cuda()
w = torch.randn(600, 512, generator=g).cuda()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
def run():
    rows, h = Q.add_rms_norm_int8(x, r, w[0])
    return Q.int8_linear(rows, Q.quantize_rows(w)), Q.dequantize_rows(rows), h
with torch.cuda.graph(graph):
    out = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, run()))
"""


@pytest.mark.parametrize("rows", [1, 40, 300, 3000])
def test_the_first_call_of_a_process_may_be_a_captured_one(rows):
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.format(rows=rows)], cwd=B.REPO, timeout=300, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]


def test_two_streams_at_once():
    sets = [boundary_inputs(100, s) for s in (50, 70)]
    want = [boundary(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(boundary(*sets[i]))
    torch.cuda.synchronize()
    for w, many in zip(want, got):
        for g in many:
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
