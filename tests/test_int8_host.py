"""The 8-bit linear path without a GPU: refusals, row layouts, devices, and that the 64-bit reference's checks can fail.
No kernel is launched here."""
import pytest
import torch

from mamba_tp_lite_b200 import _lib as L
from mamba_tp_lite_b200 import int8 as Q
from tests import int8_ref as R
from tests.test_logprobs_host import Recorder, _refused

F32, BF = torch.float32, torch.bfloat16


def rows(r=4, c=16, seed=0):
    return torch.randn(r, c, generator=torch.Generator().manual_seed(seed))


def plain(y):
    """Codes and scales of 64-bit rows."""
    scale = (y.abs().amax(-1, keepdim=True).clamp(min=1e-8) / 127).float()
    return torch.round(y / scale.double()).clamp(-127, 127).to(torch.int8), scale.squeeze(-1)


# ------------------------------------------------------------------ the reference
def test_reference_takes_the_plain_form_and_refuses_its_neighbours():
    y = rows(6, 200).double()
    y[3] = 0
    codes, scale = plain(y)
    R.check_rows(codes, scale, y)
    off = codes.clone()
    off[2, 5] += 1
    with pytest.raises(AssertionError, match="codes"):
        R.check_rows(off, scale, y)
    for factor in (1 + 2.0 ** -22, 1 - 2.0 ** -22):
        with pytest.raises(AssertionError, match="scale"):
            R.check_rows(codes, scale * factor, y)
    y[1, 7] = float("inf")
    with pytest.raises(AssertionError, match="NaN"):
        R.check_rows(codes, scale, y)
    scale[1] = float("nan")
    with pytest.raises(AssertionError, match="not finite"):
        R.check_rows(codes, scale, y)


def test_reference_norm_and_product():
    x, w = rows(3, 40).double(), rows(1, 40, 1)[0].double()
    want = torch.nn.functional.rms_norm(x, (40,), w, float(torch.tensor(1e-5)))
    torch.testing.assert_close(R.norm(x, w, 1e-5), want, rtol=1e-12, atol=1e-12)
    a = torch.full((2, 131071), -128, dtype=torch.int8)
    assert (R.sums(a, a) == 2147467264).all() and 2147467264 < 2 ** 31
    codes, scale = plain(x)
    wc, ws = plain(rows(5, 40, 2).double())
    got = R.linear(codes, scale, wc, ws, None, F32)
    want = (codes.double() * scale.double()[:, None]) @ (wc.double() * ws.double()[:, None]).T
    torch.testing.assert_close(got.double(), want, rtol=4 * R.U, atol=1e-12)


# ------------------------------------------------------------------ refusals
def test_no_cpu_path():
    x = rows()
    r = Q.Int8Rows(*plain(x.double()))
    for call in (lambda: Q.quantize_rows(x), lambda: Q.dequantize_rows(r), lambda: Q.rms_norm_int8(x, x[0]),
                 lambda: Q.add_rms_norm_int8(x, x, x[0]), lambda: Q.int8_linear(r, r)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_arguments(monkeypatch):
    rec = Recorder(monkeypatch)
    x, w = rows(), torch.ones(16)
    r = Q.Int8Rows(*plain(x.double()))
    far, wide = torch.empty(16, device="meta"), torch.randn(5, 32)
    refused = [
        (TypeError, "dtype", lambda: Q.quantize_rows(x.double())),
        (TypeError, "dtype", lambda: Q.quantize_rows(x.to(torch.int32))),
        (ValueError, "last dimension", lambda: Q.quantize_rows(torch.tensor(1.0))),
        (ValueError, "last dimension", lambda: Q.quantize_rows(torch.empty(3, 0))),
        (ValueError, "last dimension", lambda: Q.quantize_rows(torch.empty(1, 131072))),
        (ValueError, "rows", lambda: Q.quantize_rows(torch.empty(1).expand(1 << 31, 1))),
        (TypeError, "dtype", lambda: Q.dequantize_rows(r, torch.float64)),
        (TypeError, "int8 codes", lambda: Q.dequantize_rows(Q.Int8Rows(r.codes.float(), r.scale))),
        (TypeError, "int8 codes", lambda: Q.dequantize_rows(Q.Int8Rows(r.codes.view(torch.uint8), r.scale))),
        (TypeError, "float32 scales", lambda: Q.dequantize_rows(Q.Int8Rows(r.codes, r.scale.bfloat16()))),
        (ValueError, "scales of shape", lambda: Q.dequantize_rows(Q.Int8Rows(r.codes, r.scale[:3]))),
        (ValueError, "scales of shape", lambda: Q.dequantize_rows(Q.Int8Rows(r.codes, r.scale[:, None]))),
        (ValueError, "scales on", lambda: Q.dequantize_rows(Q.Int8Rows(r.codes, torch.empty(4, device="meta")))),
        (ValueError, "weight has shape", lambda: Q.rms_norm_int8(x, w[:15])),
        (ValueError, "weight is on", lambda: Q.rms_norm_int8(x, far)),
        (TypeError, "dtype", lambda: Q.rms_norm_int8(x, w.double())),
        (ValueError, "eps", lambda: Q.rms_norm_int8(x, w, -1e-5)),
        (ValueError, "eps", lambda: Q.rms_norm_int8(x, w, float("nan"))),
        (ValueError, "residual has shape", lambda: Q.add_rms_norm_int8(x, x[:3], w)),
        (ValueError, "residual is on", lambda: Q.add_rms_norm_int8(x, torch.empty(4, 16, device="meta"), w)),
        (TypeError, "dtype", lambda: Q.add_rms_norm_int8(x, x.double(), w)),
        (ValueError, "one stride", lambda: Q.add_rms_norm_int8(x, rows(16, 4).T, w, inplace=True)),
        (ValueError, "one stride", lambda: Q.add_rms_norm_int8(x, rows(1, 16).expand(4, 16), w, inplace=True)),
        (ValueError, "one stride", lambda: Q.add_rms_norm_int8(x.view(2, 2, 16), rows(6, 16).view(2, 3, 16)[:, 1:], w, inplace=True)),
        (ValueError, "share memory", lambda: Q.add_rms_norm_int8(x, x, w, inplace=True)),
        (ValueError, "share memory", lambda: Q.add_rms_norm_int8(x[:3], x[1:], w, inplace=True)),
        (ValueError, "share memory", lambda: Q.add_rms_norm_int8(rows(), x, x[3], inplace=True)),
        (ValueError, "share memory", lambda: Q.add_rms_norm_int8(wide[:, :16], wide[:, 15:31], w, inplace=True)),
        (ValueError, "share memory", lambda: Q.add_rms_norm_int8(wide[1:, :16], wide.as_strided((4, 16), (32, 1), 24), w, inplace=True)),
        (ValueError, "do not fit", lambda: Q.int8_linear(r, Q.Int8Rows(r.codes[:, :15], r.scale))),
        (ValueError, "do not fit", lambda: Q.int8_linear(r, Q.Int8Rows(r.codes[0], r.scale[0]))),
        (ValueError, "weight is on", lambda: Q.int8_linear(r, Q.Int8Rows(torch.empty(4, 16, device="meta", dtype=torch.int8),
                                                                        torch.empty(4, device="meta")))),
        (ValueError, "bias has shape", lambda: Q.int8_linear(r, r, w)),
        (ValueError, "bias is on", lambda: Q.int8_linear(r, r, far[:4])),
        (TypeError, "dtype", lambda: Q.int8_linear(r, r, w[:4].double())),
        (TypeError, "dtype", lambda: Q.int8_linear(r, r, dtype=torch.int32)),
    ]
    for error, text, call in refused:
        with pytest.raises(error, match=text):
            call()
    assert not rec.calls


def test_in_place_beside_x_and_weight_in_one_buffer(monkeypatch):
    rec = Recorder(monkeypatch)
    wide, w = torch.randn(4, 48), torch.randn(32)
    for x, res, weight in [(wide[:, :16], wide[:, 16:32], w[:16]), (wide[:, 32:], wide[:, :16], w[16:]), (wide[:2, :16], wide[2:, :16], w[:16]),
                           (wide[:0, :16], wide[:0, :16], w[:16])]:
        assert Q.add_rms_norm_int8(x, res, weight, inplace=True)[1] is res
    assert len(rec.calls) == 4


def test_in_place_is_seen_by_a_backward_pass(monkeypatch):
    Recorder(monkeypatch)
    res, scale = rows(), torch.ones(16, requires_grad=True)
    y = res * scale  # keeps res
    with torch.no_grad():
        Q.add_rms_norm_int8(rows(), res, torch.ones(16), inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_are_refused(monkeypatch):
    rec = Recorder(monkeypatch)
    x, w = rows(), torch.ones(16)
    r = Q.Int8Rows(*plain(x.double()))
    leaf = lambda t: t.clone().requires_grad_()
    calls = [lambda f: Q.quantize_rows(f(x)), lambda f: Q.dequantize_rows(Q.Int8Rows(r.codes, f(r.scale))),
             lambda f: Q.rms_norm_int8(f(x), w), lambda f: Q.rms_norm_int8(x, f(w)), lambda f: Q.add_rms_norm_int8(f(x), x, w),
             lambda f: Q.add_rms_norm_int8(x, f(x), w), lambda f: Q.int8_linear(Q.Int8Rows(r.codes, f(r.scale)), r),
             lambda f: Q.int8_linear(r, Q.Int8Rows(r.codes, f(r.scale))), lambda f: Q.int8_linear(r, r, f(w[:4]))]
    for call in calls:
        with pytest.raises(RuntimeError, match="no gradient"):
            call(leaf)
    with torch.autograd.forward_ad.dual_level():
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))
    assert not rec.calls
    with torch.no_grad():
        for call in calls:
            call(leaf)
    assert len(rec.calls) == len(calls)


def test_c_entry_points_refuse_bad_arguments():
    """Host checks, before any CUDA call: the pointers are never used."""
    p, big = 4096, 1 << 31
    q = lambda x=p, dt=L.F32, ld=16, r=4, c=16, o=p, ldo=16, s=p: ("mtp_quantize_rows", x, dt, ld, r, c, o, ldo, s, None)
    d = lambda x=p, ld=16, s=p, r=4, c=16, o=p, dt=L.F32, ldo=16: ("mtp_dequantize_rows", x, ld, s, r, c, o, dt, ldo, None)
    n = lambda x=p, xt=L.F32, ldx=16, h=p, ht=L.F32, ldh=16, o=p, ldo=16, r=4, c=16, w=p, wt=L.F32, eps=1e-5, q=p, ldq=16, s=p: (
        "mtp_rmsnorm_int8", x, xt, ldx, h, ht, ldh, o, ldo, r, c, w, wt, eps, q, ldq, s, None)
    m = lambda a=p, lda=16, s=p, M=4, K=16, w=p, ldw=16, ws=p, N=8, b=None, bt=0, o=p, dt=L.BF16, ldo=8: (
        "mtp_int8_linear", a, lda, s, M, K, w, ldw, ws, N, b, bt, o, dt, ldo, None)
    for f in (q, d, n):
        for bad in (dict(r=-1), dict(r=big), dict(c=0), dict(c=131072)):
            _refused(*f(**bad), text="rows must be")
    for bad in (q(dt=3), d(dt=-1), n(xt=9), n(ht=9), n(wt=9), m(dt=5), m(b=p, bt=4)):
        _refused(*bad, text="dtype must be")
    for bad in (q(x=None), q(o=None), q(s=None), d(x=None), d(s=None), d(o=None), n(x=None), n(o=None), n(w=None), n(q=None), n(s=None),
                m(a=None), m(s=None), m(w=None), m(ws=None), m(o=None)):
        _refused(*bad, text="null pointer")
    for bad in (q(ld=15), q(ldo=15), q(ld=-16), d(ld=15), d(ldo=0), n(ldx=15), n(ldh=15), n(ldo=15), n(ldq=15), m(lda=15), m(ldw=15),
                m(ldo=7)):
        _refused(*bad, text="leading dimensions")
    for eps in (-1.0, float("nan")):
        _refused(*n(eps=eps), text="eps")
    for bad in (dict(M=-1), dict(N=-1), dict(K=0), dict(K=131072)):
        _refused(*m(**bad), text="must")
    lib = L.load()
    for name, *args in (q(x=None, r=0), d(x=None, r=0), n(x=None, r=0), m(a=None, M=0), m(w=None, N=0)):
        assert getattr(lib, name)(*args) == L.MTP_OK  # nothing to do


# ------------------------------------------------------------------ calls, on a library that only records them
def test_every_call_is_made_on_the_device_of_its_tensors(monkeypatch):
    rec = Recorder(monkeypatch)
    x, w = rows(), torch.ones(16)
    r = Q.Int8Rows(*plain(x.double()))
    Q.quantize_rows(x), Q.dequantize_rows(r), Q.rms_norm_int8(x, w), Q.add_rms_norm_int8(x, x, w), Q.int8_linear(r, r)
    assert [c[0] for c in rec.calls] == ["mtp_quantize_rows", "mtp_dequantize_rows", "mtp_rmsnorm_int8", "mtp_rmsnorm_int8",
                                         "mtp_int8_linear"]
    assert all(depth == 1 for _, _, depth in rec.calls)


def test_strides(monkeypatch):
    """What is passed of strided, copied and single rows."""
    rec = Recorder(monkeypatch)
    x = rows(6, 40)
    Q.quantize_rows(x[:, 4:24])
    name, args, _ = rec.calls.pop()
    assert args[:5] == (x[:, 4:24].data_ptr(), L.F32, 40, 6, 20) and args[6] == 32  # codes on 16-byte boundaries
    r = Q.quantize_rows(x.view(2, 3, 40)[:, 1:])  # no common stride: copied
    assert r.codes.shape == (2, 2, 40) and r.codes.stride() == (96, 48, 1) and r.scale.shape == (2, 2)
    assert rec.calls.pop()[1][2:5] == (40, 4, 40)
    Q.quantize_rows(x.T)
    assert rec.calls.pop()[1][2:5] == (6, 40, 6)
    Q.quantize_rows(x[:1, :8])
    assert rec.calls.pop()[1][2:5] == (8, 1, 8)
    Q.quantize_rows(x[0].expand(5, 40))
    assert rec.calls.pop()[1][2:5] == (40, 5, 40)
    res = rows(6, 64, 1)
    _, h = Q.add_rms_norm_int8(x, res[:, :40], torch.ones(40), inplace=True)
    args = rec.calls.pop()[1]
    assert args[3:8] == (res.data_ptr(), L.F32, 64, res.data_ptr(), 64) and h.data_ptr() == res.data_ptr()
    _, h = Q.add_rms_norm_int8(x, res[:, :40], torch.ones(80)[::2])
    args = rec.calls.pop()[1]
    assert args[3:8] == (res.data_ptr(), L.F32, 64, h.data_ptr(), 40) and h.is_contiguous()
    codes = torch.zeros(6, 48, dtype=torch.int8)
    y = Q.int8_linear(Q.Int8Rows(codes[:, :40], torch.ones(12)[::2]), Q.Int8Rows(codes[:5, 8:], torch.ones(5)))
    args = rec.calls.pop()[1]
    assert args[1] == 48 and args[3:5] == (6, 40) and args[6] == 48 and args[8] == 5 and y.shape == (6, 5)


def test_a_model_keeps_its_parameters_and_leaves_the_one_launch_step(monkeypatch):
    from mamba_tp_lite_b200 import _decode
    from mamba_tp_lite_b200.config import MambaConfig
    from mamba_tp_lite_b200.model import MambaLM

    rec = Recorder(monkeypatch)
    lm = MambaLM(MambaConfig(d_model=64, n_layer=2, vocab_size=64, dt_rank=8)).bfloat16()
    names = list(lm.state_dict())
    assert _decode.supported(lm) is None
    lm.quantize_linears()
    assert [c[0] for c in rec.calls] == ["mtp_quantize_rows"] * 4 and not any(c[1][0] is None for c in rec.calls)
    for layer in lm.layers:
        (i, o), m = layer.mixer._int8, layer.mixer
        assert i.codes.shape == m.in_proj.weight.shape and o.codes.shape == m.out_proj.weight.shape
    assert list(lm.state_dict()) == names and _decode.supported(lm) == "int8 linears"
    lm.quantize_linears(False)
    assert _decode.supported(lm) is None and all(layer.mixer._int8 is None for layer in lm.layers)
