"""The operators on logits against their 64-bit definitions (logits_ref.py, which derives every bound used here)."""
import numpy as np
import pytest
import torch

from mamba_tp_lite_b200 import _lib as L
from mamba_tp_lite_b200 import logprobs as P
from mamba_tp_lite_b200 import quant_eval
from mamba_tp_lite_b200.checkpoint import random_init_state_dict
from mamba_tp_lite_b200.config import MambaConfig
from mamba_tp_lite_b200.model import MambaLM
from mamba_tp_lite_b200.tp_model import TPMambaLM
from tests import logits_ref as R
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu

F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16
LOW = {F32: torch.finfo(F32).min, BF: torch.finfo(BF).min, F16: torch.finfo(F16).min}


def make(rows, v, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, v, generator=g) * scale).to(dtype).to(dev())


def f64(x):
    return x.detach().double().cpu().numpy()


def close(got, want, bound, what=""):
    """|got - want| <= bound where want is finite; the same infinities and NaN elsewhere.  Results are fp32 (or
    smaller): from 2^128 - 2^103 on, half a step past the largest fp32, a value rounds to infinity (the lowest fp32
    logit divided by a temperature below 1 is one)."""
    got = f64(got) if isinstance(got, torch.Tensor) else got
    want = np.where(np.abs(want) >= 2.0 ** 128 - 2.0 ** 103, np.copysign(np.inf, want), want)
    bound = np.broadcast_to(bound, want.shape)
    fin = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=what)
    np.testing.assert_array_equal(got[np.isinf(want)], want[np.isinf(want)], err_msg=what)
    err = np.abs(got[fin] - want[fin])
    worst = (err / bound[fin]).max() if err.size else 0.0
    assert worst <= 1.0, f"{what}: error {err.max()} is {worst} of its bound"


def targets_for(rows, v, seed=0):
    t = torch.randint(0, v, (rows,), generator=torch.Generator().manual_seed(seed + 7))
    if rows > 2:
        t[1] = -1
    return t.to(dev())


def check_forward(x, t, k, temperature=1.0, entropy=True):
    """x [rows, V] as the call gets it (any layout of two dimensions)."""
    r = P.token_logprobs(x, t, top_k=k, temperature=temperature, entropy=entropy)
    xa = f64(x)
    want = R.token_logprob(xa, t.cpu().numpy(), temperature)
    close(r.logprob, want, R.logprob_bound(xa, want, temperature), "logprob")
    if entropy:
        close(r.entropy, R.entropy(xa, temperature), R.entropy_bound(xa, temperature), "entropy")
    else:
        assert r.entropy is None
    if k:
        ids = R.top(xa, k)
        np.testing.assert_array_equal(r.top_ids.cpu().numpy(), ids)
        lp = np.take_along_axis(R.log_probs(xa, temperature), ids, 1)
        close(r.top_logprobs, lp, R.logprob_bound(xa, lp, temperature), "top_logprobs")
    else:
        assert r.top_ids is None and r.top_logprobs is None
    return r


# ------------------------------------------------------------------ forward
SIZES = [(1, 1), (3, 2), (5, 7), (4, 63), (9, 257), (2, 1000), (33, 1001), (1, 50280), (7, 50277), (2, 131072), (3, 70001)]


@pytest.mark.parametrize("rows,v", SIZES)
@pytest.mark.parametrize("dtype", [F32, BF, F16])
def test_token_logprobs_match_the_definition(rows, v, dtype):
    x = make(rows, v, dtype, rows * 31 + v)
    t = targets_for(rows, v)
    for k in sorted({0, 1, min(5, v), min(64, v), min(128, v)}):
        check_forward(x, t, k)


@pytest.mark.parametrize("temperature", [0.3, 2.5])
@pytest.mark.parametrize("entropy", [True, False])
def test_token_logprobs_temperature(temperature, entropy):
    x = make(12, 3001, BF, 5)
    check_forward(x, targets_for(12, 3001), 10, temperature, entropy)


def test_token_logprobs_without_targets():
    x = make(4, 500, F32, 6)
    r = P.token_logprobs(x, top_k=3)
    assert r.logprob is None and r.top_ids.shape == (4, 3)
    close(r.entropy, R.entropy(f64(x)), R.entropy_bound(f64(x)))


@pytest.mark.parametrize("rows", [148, 1200, 5000])
@pytest.mark.parametrize("v", [24, 1003])
def test_token_logprobs_many_rows(rows, v):
    check_forward(make(rows, v, BF, rows), targets_for(rows, v), 4)


WARP_ROWS = 2500  # short rows in such numbers go a warp each


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("v", [1, 9, 130, 1003, 3000])
def test_short_rows_in_large_numbers(dtype, v):
    """Forward, gradient and distillation of rows that a warp takes each, with rows where a softmax goes
    wrong easily among them."""
    x = make(WARP_ROWS, v, dtype, v)
    if v >= 40:
        x[:16] = special_rows(v, dtype)
        x[-16:] = x[:16]
    t = targets_for(WARP_ROWS, v)
    for k in sorted({0, 1, min(7, v), min(64, v), min(128, v)}):
        check_forward(x, t, k, 0.8)
    g = torch.linspace(0.5, 1.5, WARP_ROWS, device=dev())
    h = torch.linspace(-1, 0.9, WARP_ROWS, device=dev())
    for heads in (2, 1):
        leaf = x.detach().requires_grad_()
        r = P.token_logprobs(leaf, t)
        outs, grads = [r.logprob, r.entropy][:heads], [g, h][:heads]
        (grad,) = torch.autograd.grad(outs, [leaf], grads)
        check_grad(x, t, g, h if heads == 2 else torch.zeros_like(h), grad)
    x = make(WARP_ROWS, v, dtype, v)
    ids, vals = teacher_for(x, min(20, v))
    ids[3] = -1
    ids[4] = ids[4, 0].clone()
    loss, grad = P.distill_topk_loss_and_grad(x, ids, vals, g)
    check_distill(x, ids, vals, g, loss, grad)
    leaf = x.detach().requires_grad_()
    loss = P.distill_topk_loss(leaf, ids, vals)
    (grad,) = torch.autograd.grad([loss], [leaf], [g])
    check_distill(x, ids, vals, g, loss, grad)


@pytest.mark.parametrize("rows,v,dtype", [(160, 60000, F32), (150, 131071, BF), (20, 131072, F32), (149, 30001, F32)])
def test_long_rows_shared_by_clusters(rows, v, dtype):
    x = make(rows, v, dtype, 4)
    t = targets_for(rows, v)
    check_forward(x, t, 33)
    ids, vals = teacher_for(x, 40)
    w = torch.linspace(0.5, 1.5, rows, device=dev())
    loss, grad = P.distill_topk_loss_and_grad(x, ids, vals, w)
    check_distill(x, ids, vals, w, loss, grad)


LAYOUTS = {
    "shifted": lambda x: x.view(4, 6, -1)[:, :-1],
    "cut": lambda x: x.view(4, 6, -1)[..., :-3],
    "cut_front": lambda x: x.view(4, 6, -1)[..., 1:],
    "cut_and_shifted": lambda x: x.view(4, 6, -1)[:, 1:, 5:-2],
    "three_strides": lambda x: x.view(2, 3, 4, -1)[:, :2, :3, :-1],
    "every_other": lambda x: x[::2],
    "columns": lambda x: x.t().contiguous().t(),
    "expanded": lambda x: x[:1].expand(6, -1),
    "transposed": lambda x: x.view(4, 6, -1).transpose(0, 1),
    "one": lambda x: x[3],
}


@pytest.mark.parametrize("name", LAYOUTS)
@pytest.mark.parametrize("dtype", [F32, BF])
def test_layouts_give_the_same_as_a_dense_copy(name, dtype):
    """Forward and gradient of strided logits against the definition on their dense copy."""
    x = LAYOUTS[name](make(24, 1013, dtype, 11))
    lead = x.shape[:-1]
    rows = x.numel() // x.shape[-1]
    dense = x.reshape(rows, -1).contiguous()
    t = targets_for(rows, dense.shape[1])
    r = P.token_logprobs(x, t.view(lead), top_k=6)
    assert r.logprob.shape == lead and r.top_ids.shape == (*lead, 6)
    xa = f64(dense)
    want = R.token_logprob(xa, t.cpu().numpy())
    close(r.logprob.reshape(rows), want, R.logprob_bound(xa, want))
    np.testing.assert_array_equal(r.top_ids.reshape(rows, 6).cpu().numpy(), R.top(xa, 6))
    g = torch.linspace(-1, 1, rows, device=dev())
    h = torch.linspace(0.5, -0.5, rows, device=dev())
    leaf = x.detach().requires_grad_()
    rr = P.token_logprobs(leaf, t.view(lead))
    (grad,) = torch.autograd.grad([rr.logprob, rr.entropy], [leaf], [g.view(lead), h.view(lead)])
    assert grad.shape == x.shape and grad.dtype == dtype
    check_grad(dense, t, g, h, grad.reshape(rows, -1))
    ids = r.top_ids
    loss, dg = P.distill_topk_loss_and_grad(x, ids, r.top_logprobs, g.view(lead))
    assert dg.shape == x.shape
    check_distill(dense, ids.reshape(rows, 6), r.top_logprobs.reshape(rows, 6), g, loss.reshape(rows),
                  dg.reshape(rows, -1))


def special_rows(v, dtype):
    """Rows where a softmax goes wrong easily, v >= 40."""
    x = make(16, v, F32, 3)
    inf = float("inf")
    x[0] = -inf                      # nothing left
    x[1] = -inf
    x[1, v - 1] = 2.0                # one token left
    x[2, 1::2] = -inf                # every other token masked
    x[3, 5:] = LOW[dtype]            # masked with the type's lowest value
    x[4] = LOW[dtype]                # nothing but the lowest value: uniform
    x[5] = 0.0                       # all equal
    x[6] = 0.0
    x[6, ::3] = -0.0                 # equal, of both signs
    x[7] = torch.arange(v) * 0.01    # rising
    x[8] = torch.arange(v, 0, -1) * 0.01
    x[9] = 60000.0 if dtype == F16 else 1e30
    x[9, 3] = -x[9, 3]
    x[10, 7] = inf
    x[11, 9] = float("nan")
    x[12] = float("nan")
    x[13, 2] = inf
    x[13, 3] = float("nan")
    x[13, v - 2] = float("nan")
    x[14, v // 2] += 200.0           # certain
    x[15, : v // 2] = x[15, 0]       # half of them tied
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("v", [40, 3000, 50283])
def test_special_rows(dtype, v):
    x = special_rows(v, dtype)
    for shift in (0, 3):
        t = torch.full((16,), shift, device=dev())
        t[5], t[6] = v, -3
        for k in (0, 1, 17, min(128, v)):
            check_forward(x, t, k)
    g = torch.linspace(0.5, 1.5, 16, device=dev())
    h = torch.linspace(-1, 0.9, 16, device=dev())
    t[5] = 1
    leaf = x.detach().requires_grad_()
    r = P.token_logprobs(leaf, t)
    (grad,) = torch.autograd.grad([r.logprob, r.entropy], [leaf], [g, h])
    check_grad(x, t, g, h, grad)


# ------------------------------------------------------------------ gradients
TINY = {F32: 2.0 ** -126, BF: 2.0 ** -126, F16: 2.0 ** -25}


def check_grad(x, t, g, h, grad, temperature=1.0):
    xa = f64(x)
    want, mag = R.token_logprobs_grad(xa, t.cpu().numpy(), f64(g), f64(h), temperature)
    bad = ~np.isfinite(R.log_probs(xa, temperature).max(-1)) & ~np.isneginf(xa).all(-1)
    got = f64(grad)
    assert np.isnan(got[bad]).all()
    ok = ~bad
    # the largest magnitudes of a row's terms, so that the bound of an element is never below the rounding of a sum
    close(got[ok], want[ok], R.grad_bound(xa[ok], want[ok], mag[ok], torch.finfo(grad.dtype).eps, TINY[grad.dtype],
                                          temperature), "gradient")


@pytest.mark.parametrize("rows,v", [(1, 1), (3, 2), (5, 63), (33, 1001), (4, 50280), (7, 50277), (2, 131072)])
@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("which", ["both", "logprob", "entropy"])
def test_token_logprobs_gradient_matches_the_formula(rows, v, dtype, which):
    x = make(rows, v, dtype, rows + v)
    t = targets_for(rows, v)
    g = torch.linspace(0.5, 1.5, rows, device=dev())
    h = torch.linspace(-1, 0.9, rows, device=dev())
    leaf = x.detach().requires_grad_()
    r = P.token_logprobs(leaf, t, temperature=1.25)
    outs, grads = [r.logprob, r.entropy], [g, h]
    if which == "logprob":
        outs, grads, h = outs[:1], grads[:1], torch.zeros_like(h)
    if which == "entropy":
        outs, grads, g = outs[1:], grads[1:], torch.zeros_like(g)
    (grad,) = torch.autograd.grad(outs, [leaf], grads)
    check_grad(x, t, g, h, grad, 1.25)


def test_gradients_match_differences():
    """fp32 kernels' own forward along a direction u: (f(x + s u) - f(x - s u)) / 2s against <grad, u>.
    f is a sum over 6 rows; each value is known to its bound, so the difference to twice their sum / 2s, and the third
    derivative along |u| <= 1 of a log partition function and an entropy is at most 2 and 2 + 6 H: s^2 / 6 of it."""
    x = make(6, 1500, F32, 1)
    t = targets_for(6, 1500)
    ids = torch.randint(0, 1500, (6, 20), device=dev())
    vals = make(6, 20, F32, 2)
    g = torch.linspace(0.5, 1.5, 6, device=dev())
    h = torch.linspace(-1, 0.9, 6, device=dev())
    u = torch.rand(6, 1500, generator=torch.Generator().manual_seed(3)).to(dev()) * 2 - 1
    s = 2.0 ** -6
    xa = f64(x)
    ent = R.entropy(xa)

    def f_tok(y):
        r = P.token_logprobs(y, t)
        return (g * r.logprob + h * r.entropy).double().sum().item()

    def f_dis(y):
        return (g * P.distill_topk_loss(y, ids, vals)).double().sum().item()

    leaf = x.detach().requires_grad_()
    r = P.token_logprobs(leaf, t)
    (gt,) = torch.autograd.grad([r.logprob, r.entropy], [leaf], [g, h])
    (gd,) = torch.autograd.grad([P.distill_topk_loss(leaf, ids, vals)], [leaf], [g])
    want = R.token_logprob(xa, t.cpu().numpy())
    noise = (f64(g) * R.logprob_bound(xa, want) + np.abs(f64(h)) * R.entropy_bound(xa)).sum() * 2 / (2 * s)
    curve = ((f64(g) * 2 + np.abs(f64(h)) * (2 + 6 * ent)) * s * s / 6).sum()
    moved = (f_tok(x + s * u) - f_tok(x - s * u)) / (2 * s)
    # x + s u is rounded to fp32: the step is off by at most half a step of |x| <= 16 on each side
    step = 2.0 ** -21 / s * (f64(g) * 2 + np.abs(f64(h)) * 20).sum()
    assert abs(moved - (gt.double() * u.double()).sum().item()) <= noise + curve + step
    moved = (f_dis(x + s * u) - f_dis(x - s * u)) / (2 * s)
    q, log_q = R.teacher(ids.cpu().numpy(), f64(vals))
    lp = np.take_along_axis(R.log_probs(xa), ids.cpu().numpy(), 1)
    noise = (f64(g) * distill_bound(xa, q, log_q, lp)).sum() * 2 / (2 * s)
    assert abs(moved - (gd.double() * u.double()).sum().item()) <= noise + curve + step


def test_second_derivative_is_refused():
    x = make(2, 50, F32).requires_grad_()
    r = P.token_logprobs(x, targets_for(2, 50))
    (grad,) = torch.autograd.grad([r.logprob.sum()], [x], create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_unused_rows_get_a_zero_gradient_whatever_they_hold():
    x = make(4, 100, F32)
    x[1] = float("nan")
    x[2, 4] = float("inf")
    leaf = x.detach().requires_grad_()
    r = P.token_logprobs(leaf, torch.tensor([3, -1, 5, 6], device=dev()))
    w = torch.tensor([1.0, 1.0, 0.0, 1.0], device=dev())
    (grad,) = torch.autograd.grad([r.logprob], [leaf], [w])
    assert (grad[1] == 0).all() and (grad[2] == 0).all() and (grad[0] != 0).all()
    ids = torch.zeros(4, 2, dtype=torch.int64, device=dev())
    _, grad = P.distill_topk_loss_and_grad(x, ids, torch.zeros(4, 2, device=dev()),
                                           torch.tensor([1.0, 0.0, 0.0, 1.0], device=dev()))
    assert (grad[1] == 0).all() and (grad[2] == 0).all() and (grad[0] != 0).all()


# ------------------------------------------------------------------ distillation
def distill_bound(xa, q, log_q, lp, temperature=1.0):
    """A sum of q (log q - log p): q and log q from at most 128 terms, each to 8 u + 2^-22 + 2 u |log q|; the log
    probabilities to their bound; the sum of 128 terms to 16 u."""
    lq = np.where(q > 0, np.abs(log_q), 0)
    lpa = np.where((q > 0) & np.isfinite(lp), np.abs(lp), 0)
    b = R.logprob_bound(xa, np.where(np.isfinite(lp), lp, 0), temperature)
    rel = 16 * R.U + 2.0 ** -21 + 4 * R.U * (lq + 2)
    return (q * (b + (lq + lpa + 1) * (rel + 16 * R.U))).sum(-1) + 2.0 ** -40


def check_distill(x, ids, vals, w, loss, grad, temperature=1.0):
    xa, ia, va = f64(x), ids.cpu().numpy(), f64(vals)
    v = xa.shape[1]
    q, log_q = R.teacher(ia, va, temperature)
    lp = np.take_along_axis(R.log_probs(xa, temperature), np.clip(ia, 0, v - 1), 1)
    want = R.distill_loss(xa, ia, va, temperature)
    close(loss, want, distill_bound(xa, q, log_q, lp, temperature), "loss")
    if grad is None:
        return
    bad = ((ia >= v) & (q > 0)).any(-1) & (f64(w) != 0)
    got = f64(grad)
    assert np.isnan(got[bad]).all()
    ok = ~bad
    want, mag = R.distill_grad(xa[ok], np.where(ia[ok] >= v, 0, ia[ok]), np.where(ia[ok] >= v, -np.inf, va[ok]),
                               f64(w)[ok], temperature)
    want = np.where((f64(w)[ok] == 0)[:, None], 0.0, want)
    close(got[ok], want, R.grad_bound(xa[ok], want, mag, torch.finfo(grad.dtype).eps, TINY[grad.dtype], temperature),
          "gradient")


def teacher_for(x, k, seed=0):
    rows, v = x.shape
    g = torch.Generator().manual_seed(seed)
    noisy = x.float().cpu() + torch.randn(rows, v, generator=g)
    top = noisy.topk(k, -1)
    return top.indices.to(dev()), top.values.to(dev())


@pytest.mark.parametrize("rows,v,k", [(1, 1, 1), (3, 2, 2), (5, 63, 9), (33, 1001, 64), (4, 50280, 128), (7, 50277, 31),
                                      (2, 131072, 64), (1300, 130, 20)])
@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_distillation_matches_the_formula(rows, v, k, dtype, temperature):
    x = make(rows, v, dtype, rows + v)
    ids, vals = teacher_for(x, k)
    w = torch.linspace(0.5, 1.5, rows, device=dev())
    loss = P.distill_topk_loss(x, ids, vals, temperature=temperature)
    check_distill(x, ids, vals, w, loss, None, temperature)
    loss, grad = P.distill_topk_loss_and_grad(x, ids, vals, w, temperature=temperature)
    check_distill(x, ids, vals, w, loss, grad, temperature)
    leaf = x.detach().requires_grad_()
    loss = P.distill_topk_loss(leaf, ids, vals, temperature=temperature)
    (grad,) = torch.autograd.grad([loss], [leaf], [w])
    check_distill(x, ids, vals, w, loss, grad, temperature)


@pytest.mark.parametrize("vdt", [F32, BF, F16])
def test_distillation_teacher_entries(vdt):
    """Unused entries, equal ids, ids out of range, rows without a used entry, weights of zero."""
    x = make(10, 300, BF, 4)
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, 300, (10, 12), generator=g)
    vals = (torch.randn(10, 12, generator=g) * 2).to(vdt)
    ids[0] = -1                                # nothing used
    vals[1] = float("-inf")                    # nothing used
    ids[2, 3:] = -7                            # padded
    vals[3, ::2] = float("-inf")
    ids[4] = 17                                # one token twelve times
    ids[5, 4] = ids[5, 9] = ids[5, 0]
    ids[6, 2] = 300                            # out of range and used
    ids[7, 2], vals[7, 2] = 1 << 40, float("-inf")  # out of range, not used
    vals[8, 0] = 80.0                          # certain
    ids, vals = ids.to(dev()), vals.to(dev())
    w = torch.linspace(-0.5, 1.5, 10, device=dev())
    w[9] = 0.0
    loss, grad = P.distill_topk_loss_and_grad(x, ids, vals, w)
    check_distill(x, ids, vals, w, loss, grad)
    assert loss[0] == 0 and loss[1] == 0 and (grad[0] == 0).all() and (grad[9] == 0).all()
    leaf = x.detach().requires_grad_()
    loss = P.distill_topk_loss(leaf, ids, vals)
    (grad,) = torch.autograd.grad([loss], [leaf], [w])
    check_distill(x, ids, vals, w, loss, grad)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
def test_distillation_special_student_rows(dtype):
    x = special_rows(3000, dtype)[:10]
    ids = torch.tensor([1, 2, 4, 2999], device=dev()).expand(10, 4)
    vals = make(10, 4, F32, 9)
    w = torch.ones(10, device=dev())
    loss, grad = P.distill_topk_loss_and_grad(x, ids, vals, w)
    assert loss[0] == float("inf") and (grad[0] == 0).all()  # probability 0 for a token the teacher gives
    check_distill(x, ids, vals, w, loss, grad)


def test_distillation_from_its_own_alternatives_is_zero():
    """The teacher recorded from the same logits, all of the vocabulary: loss and gradient vanish to their bounds."""
    x = make(9, 100, F32, 2)
    top = P.token_logprobs(x, top_k=100)
    w = torch.ones(9, device=dev())
    loss, grad = P.distill_topk_loss_and_grad(x, top.top_ids, top.top_logprobs, w)
    check_distill(x, top.top_ids, top.top_logprobs, w, loss, grad)
    assert loss.abs().max() < 1e-4


# ------------------------------------------------------------------ from hidden states
def score_inputs(rows, v, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(rows, k, generator=g).to(dtype).to(dev())
    w = (torch.randn(v, k, generator=g) * (2.0 / k ** 0.5)).to(dtype).to(dev())
    return h, w


def check_score(h, w, t, r, temperature=1.0):
    """Logits from products summed in fp32: each off by at most (K + 32) u times the sum of |h| |w| (a bound that the
    tensor core's own order and truncating alignment, at most one bit a step more, meets with a factor of 2); a log
    probability and an entropy then move by at most twice the largest such change, and (1 + their spread) of it."""
    ha, wa = f64(h), f64(w)
    x = ha @ wa.T
    dz = 2 * (ha.shape[1] + 32) * R.U * (np.abs(ha) @ np.abs(wa).T).max(-1) / temperature
    # random signs: a chain of K roundings grows as sqrt(K); the bound above is K / sqrt(K) looser than what is seen
    want = R.token_logprob(x, t.cpu().numpy(), temperature)
    close(r.logprob, want, R.logprob_bound(x, want, temperature) + 2 * dz, "logprob")
    if r.entropy is not None:
        _, _, log_s, d = R.softmax_parts(x, temperature)
        spread = np.abs(log_s[:, 0]) + 2
        close(r.entropy, R.entropy(x, temperature), R.entropy_bound(x, temperature) + 4 * dz * spread, "entropy")
    return x


@pytest.mark.parametrize("rows,v,k", [(1, 1, 8), (1, 50280, 768), (3, 17, 64), (64, 1000, 768), (65, 4097, 200),
                                      (130, 50277, 64), (300, 2049, 2048), (129, 255, 8), (128, 256, 64), (1, 300, 72),
                                      (513, 777, 328), (2000, 1030, 128)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_lm_head_logprobs_match_the_definition(rows, v, k, dtype):
    h, w = score_inputs(rows, v, k, dtype, rows + v)
    t = targets_for(rows, v)
    check_score(h, w, t, P.lm_head_logprobs(h, w, t))
    check_score(h, w, t, P.lm_head_logprobs(h, w, t, temperature=0.7, entropy=False), 0.7)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_lm_head_logprobs_alternatives_are_those_of_its_logits(dtype):
    h, w = score_inputs(70, 3001, 256, dtype)
    t = targets_for(70, 3001)
    r = P.lm_head_logprobs(h, w, t, top_k=9)
    x = check_score(h, w, t, r)
    # the logits at the chosen ids, up to their error, are the largest ones in falling order
    got = np.take_along_axis(x, r.top_ids.cpu().numpy(), 1)
    best = -np.sort(-x, -1)[:, :9]
    dz = 2 * (256 + 32) * R.U * (np.abs(f64(h)) @ np.abs(f64(w)).T).max(-1)[:, None]
    assert (np.abs(got - best) <= 2 * dz).all()
    lp = np.take_along_axis(R.log_probs(x), r.top_ids.cpu().numpy(), 1)
    close(r.top_logprobs, lp, R.logprob_bound(x, lp) + 2 * dz)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_lm_head_logprobs_strides_and_targets(dtype):
    """Hidden states and weights that are slices of wider ones, at aligned and odd offsets; a batch."""
    h, w = score_inputs(24, 500, 96, dtype, 8)
    for a, b in ((8, 88), (1, 65), (0, 63)):
        hs, ws = h.view(4, 6, 96)[..., a:b], w[:, a:b]
        t = targets_for(24, 500).view(4, 6)
        r = P.lm_head_logprobs(hs, ws, t)
        assert r.logprob.shape == (4, 6)
        check_score(hs.reshape(24, -1), ws, t.reshape(24), P.TokenLogprobs(r.logprob.view(24), r.entropy.view(24), None,
                                                                           None))
    t = torch.tensor([-1, 499, 500] + [0] * 21, device=dev())
    r = P.lm_head_logprobs(h, w, t)
    assert r.logprob[0] == 0 and torch.isnan(r.logprob[2]) and torch.isfinite(r.logprob[1])
    assert P.lm_head_logprobs(h, w).logprob is None


def test_lm_head_logprobs_non_finite_hidden_states():
    h, w = score_inputs(40, 700, 64, BF, 3)
    h[3, 5], h[20, 0] = float("nan"), float("inf")
    t = targets_for(40, 700)
    r = P.lm_head_logprobs(h, w, t)
    bad = torch.zeros(40, dtype=torch.bool, device=dev())
    bad[3] = bad[20] = True
    assert torch.isnan(r.logprob[bad]).all() and torch.isnan(r.entropy[bad]).all()
    assert torch.isfinite(r.logprob[~bad]).all() and torch.isfinite(r.entropy[~bad]).all()


def test_lm_head_logprobs_refusals():
    h, w = score_inputs(4, 50, 16, BF)
    t = targets_for(4, 50)
    with pytest.raises(TypeError):
        P.lm_head_logprobs(h.half(), w.half(), t)
    with pytest.raises(TypeError):
        P.lm_head_logprobs(h, w.float(), t)
    with pytest.raises(ValueError):
        P.lm_head_logprobs(h, w[:, :8], t)
    with pytest.raises(ValueError):
        P.lm_head_logprobs(h, w, t[:3])
    with pytest.raises(RuntimeError, match="no gradient"):
        P.lm_head_logprobs(h.detach().requires_grad_(), w, t)


# ------------------------------------------------------------------ refusals on the device
def test_refusals():
    x = make(4, 50, F32)
    t = targets_for(4, 50)
    with pytest.raises(TypeError):
        P.token_logprobs(x.double(), t)
    with pytest.raises(TypeError):
        P.token_logprobs(x, t.float())
    with pytest.raises(ValueError):
        P.token_logprobs(x, t[:3])
    with pytest.raises(ValueError):
        P.token_logprobs(x, t.cpu())
    with pytest.raises(ValueError):
        P.token_logprobs(x, t, top_k=51)
    with pytest.raises(ValueError):
        P.token_logprobs(x, t, temperature=0.0)
    with pytest.raises(ValueError):
        P.distill_topk_loss(x, t, t.float())
    with pytest.raises(TypeError):
        P.distill_topk_loss(x, t[:, None], t[:, None])
    with pytest.raises(ValueError):
        P.distill_topk_loss_and_grad(x, t[:, None], t[:, None].float(), torch.ones(3, device=dev()))


def test_empty_batches():
    x = torch.empty(0, 5, 30, device=dev(), dtype=BF)
    t = torch.empty(0, 5, dtype=torch.int64, device=dev())
    r = P.token_logprobs(x, t, top_k=3)
    assert r.logprob.shape == (0, 5) and r.top_ids.shape == (0, 5, 3)
    leaf = x.detach().requires_grad_()
    P.token_logprobs(leaf, t).logprob.sum().backward()
    assert leaf.grad.shape == x.shape
    ids = torch.empty(0, 5, 2, dtype=torch.int64, device=dev())
    loss, grad = P.distill_topk_loss_and_grad(x, ids, ids.float(), t.float())
    assert loss.shape == (0, 5) and grad.shape == x.shape
    r = P.lm_head_logprobs(torch.empty(0, 16, device=dev()), torch.randn(30, 16, device=dev()),
                           torch.empty(0, dtype=torch.int64, device=dev()))
    assert r.logprob.shape == (0,)


# ------------------------------------------------------------------ how calls are made
def test_offsets_past_32_bits():
    """More than 2^31 elements: the last rows are those a small call gives."""
    rows, v = 43000, 50280
    x = torch.zeros(rows, v, device=dev(), dtype=BF)
    tail = make(3, v, BF, 1)
    x[-3:] = tail
    t = torch.full((rows,), 17, device=dev())
    r = P.token_logprobs(x, t, top_k=2)
    small = P.token_logprobs(tail, t[-3:], top_k=2)
    assert torch.equal(r.top_ids[-3:], small.top_ids)
    xa = f64(tail)
    want = R.token_logprob(xa, t[-3:].cpu().numpy())
    close(r.logprob[-3:], want, R.logprob_bound(xa, want))
    assert (r.top_ids[:-3] == torch.tensor([0, 1], device=dev())).all()
    g = torch.ones(rows, device=dev())
    leaf = x.detach().requires_grad_()
    rr = P.token_logprobs(leaf, t)
    (grad,) = torch.autograd.grad([rr.logprob], [leaf], [g])
    check_grad(tail, t[-3:], g[-3:], torch.zeros(3, device=dev()), grad[-3:])
    del grad, rr, leaf
    ids, vals = teacher_for(tail, 5)
    loss, grad = P.distill_topk_loss_and_grad(x, torch.cat([ids[:1].expand(rows - 3, 5), ids]),
                                              torch.cat([vals[:1].expand(rows - 3, 5), vals]), g)
    check_distill(tail, ids, vals, g[-3:], loss[-3:], grad[-3:])


@pytest.mark.parametrize("rows,v,k", [(1, 50280, 5), (300, 4001, 64)])
def test_same_bits_every_time(rows, v, k):
    x = make(rows, v, BF, 3)
    t = targets_for(rows, v)
    ids, vals = teacher_for(x, k)
    w = torch.ones(rows, device=dev())
    a, b = P.token_logprobs(x, t, top_k=k), P.token_logprobs(x, t, top_k=k)
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    a, b = (P.distill_topk_loss_and_grad(x, ids, vals, w) for _ in range(2))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    h, wt = score_inputs(rows, v, 64, BF)
    a, b = P.lm_head_logprobs(h, wt, t), P.lm_head_logprobs(h, wt, t)
    assert torch.equal(a.logprob, b.logprob) and torch.equal(a.entropy, b.entropy)


def test_rows_after_the_last_stay_as_they_are():
    """Outputs of a call on the first rows of larger buffers leave the rest alone (through the C entry points)."""
    rows, v, k, ldg = 5, 333, 4, 340
    x = make(rows, v, BF, 1)
    t = targets_for(rows, v)
    lp, ent, tl = (torch.full(s, 7.0, device=dev()) for s in ((8,), (8,), (8, k)))
    st = torch.full((8, 2), 7.0, device=dev())
    ids = torch.full((8, k), 7, dtype=torch.int64, device=dev())
    L.call("mtp_token_logprobs", L.ptr(x), L.BF16, 1, rows, 0, v, v, L.ptr(t), 1.0, L.ptr(lp), L.ptr(ent), L.ptr(st), k,
           L.ptr(ids), L.ptr(tl), L.stream_ptr())
    for o in (lp, ent, st, ids, tl):
        assert (o[rows:] == 7).all()
    grad = torch.full((8, ldg), 7.0, device=dev(), dtype=BF)
    L.call("mtp_token_logprobs_bwd", L.ptr(x), L.BF16, 1, rows, 0, v, v, L.ptr(t), 1.0, L.ptr(st), L.ptr(ent), L.ptr(lp),
           L.ptr(ent), L.ptr(grad), 0, ldg, L.stream_ptr())
    assert (grad[rows:] == 7).all() and (grad[:, v:] == 7).all()
    check_grad(x, t, lp[:rows], ent[:rows], grad[:rows, :v])
    grad.fill_(7.0)
    loss = torch.full((8,), 7.0, device=dev())
    w = torch.ones(8, device=dev())
    L.call("mtp_distill_topk_grad", L.ptr(x), L.BF16, 1, rows, 0, v, v, L.ptr(ids), L.ptr(tl), L.F32, k, 1.0, None,
           L.ptr(w), L.ptr(loss), L.ptr(grad), 0, ldg, L.stream_ptr())
    assert (grad[rows:] == 7).all() and (grad[:, v:] == 7).all() and (loss[rows:] == 7).all()
    check_distill(x, ids[:rows], tl[:rows], w[:rows], loss[:rows], grad[:rows, :v])


def test_gradient_rows_of_another_alignment():
    """The C entry points take a gradient whose rows are aligned otherwise than the logits'."""
    rows, v = 6, 1000
    for dtype in (F32, BF, F16):
        x = make(rows, v, dtype, 2)
        t = targets_for(rows, v)
        r = P.token_logprobs(x, t)
        stats = torch.empty(rows, 2, device=dev())
        L.call("mtp_token_logprobs", L.ptr(x), L.dtype_code(dtype), 1, rows, 0, v, v, None, 1.0, None, None,
               L.ptr(stats), 0, None, None, L.stream_ptr())
        buf = torch.full((rows, v + 5), 7.0, device=dev(), dtype=dtype)
        grad = buf[:, 3:3 + v]
        g, h = torch.ones(rows, device=dev()), torch.full((rows,), 0.5, device=dev())
        L.call("mtp_token_logprobs_bwd", L.ptr(x), L.dtype_code(dtype), 1, rows, 0, v, v, L.ptr(t), 1.0, L.ptr(stats),
               L.ptr(r.entropy), L.ptr(g), L.ptr(h), grad.data_ptr(), 0, v + 5, L.stream_ptr())
        check_grad(x, t, g, h, grad)
        assert (buf[:, :3] == 7).all() and (buf[:, 3 + v:] == 7).all()
        ids, vals = teacher_for(x, 9)
        loss = torch.empty(rows, device=dev())
        L.call("mtp_distill_topk_grad", L.ptr(x), L.dtype_code(dtype), 1, rows, 0, v, v, L.ptr(ids), L.ptr(vals), L.F32,
               9, 1.0, None, L.ptr(g), L.ptr(loss), grad.data_ptr(), 0, v + 5, L.stream_ptr())
        check_distill(x, ids, vals, g, loss, grad)
        assert (buf[:, :3] == 7).all() and (buf[:, 3 + v:] == 7).all()


def test_two_streams_at_once_and_a_side_stream():
    x, y = make(400, 9001, BF, 1), make(500, 7001, BF, 2)
    tx, ty = targets_for(400, 9001), targets_for(500, 7001)
    h, w = score_inputs(300, 5000, 256, BF)
    th = targets_for(300, 5000)
    want = (P.token_logprobs(x, tx, top_k=8), P.token_logprobs(y, ty, top_k=3), P.lm_head_logprobs(h, w, th))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s1):
            a = P.token_logprobs(x, tx, top_k=8)
            c = P.lm_head_logprobs(h, w, th)
        with torch.cuda.stream(s2):
            b = P.token_logprobs(y, ty, top_k=3)
            d = P.lm_head_logprobs(h, w, th)
        torch.cuda.synchronize()
        for got, ref in ((a, want[0]), (b, want[1]), (c, want[2]), (d, want[2])):
            assert all(torch.equal(i, j) for i, j in zip(got, ref) if i is not None)


def test_captured_and_replayed():
    """Forward, gradient, distillation and scoring in one graph, replayed on new inputs; two graphs alive at once."""
    x = make(40, 3001, BF, 1)
    t = targets_for(40, 3001)
    ids, vals = teacher_for(x, 8)
    w = torch.ones(40, device=dev())
    h, wt = score_inputs(40, 900, 64, BF)
    th = targets_for(40, 900)

    def work():
        leaf = x.detach().requires_grad_()
        r = P.token_logprobs(leaf, t, top_k=5)
        (grad,) = torch.autograd.grad([r.logprob, r.entropy], [leaf], [w, w])
        loss, dg = P.distill_topk_loss_and_grad(x, ids, vals, w)
        s = P.lm_head_logprobs(h, wt, th)
        return [o.detach() for o in (r.logprob, r.entropy, r.top_ids, r.top_logprobs, grad, loss, dg, s.logprob, s.entropy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = work()
        graphs.append((gr, out))
    for seed in (5, 6):
        x.copy_(make(40, 3001, BF, seed))
        h.copy_(score_inputs(40, 900, 64, BF, seed)[0])
        want = work()
        for gr, out in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for gr, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


# ------------------------------------------------------------------ together, as they are used
def small_model(cls, dtype):
    cfg = MambaConfig(d_model=128, n_layer=2, vocab_size=1003, dt_rank=16)
    sd = random_init_state_dict(cfg, seed=0, dtype=dtype)
    sd["backbone.embeddings.weight"] = sd["backbone.embeddings.weight"] * 8
    if cls is MambaLM:
        return cfg, MambaLM.from_state_dict(cfg, sd, dtype, "cuda:0")
    return cfg, TPMambaLM.from_state_dict_shard(cfg, sd, 0, 1, dtype=dtype, allreduce_dtype="fp32", device="cuda:0")


@pytest.mark.parametrize("cls", [MambaLM, TPMambaLM])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_model_score(cls, dtype):
    """score() against the log probabilities of the logits that lm_head rounds to the model dtype: they differ by at
    most that rounding (half a step of the largest logit, twice) and the products' own order; the caches are the same
    and a prompt scored in two parts gives what it gives in one."""
    cfg, m = small_model(cls, dtype)
    ids = torch.randint(0, cfg.vocab_size, (3, 40), generator=torch.Generator().manual_seed(1)).to(dev())
    r, cache = m.score(ids, top_k=4)
    logits, ref_cache = m.prefill(ids)
    for a, b in zip(cache.layers, ref_cache.layers):
        assert torch.equal(a.ssm_state, b.ssm_state) and torch.equal(a.conv_state, b.conv_state)
    ref = P.token_logprobs(logits[:, :-1], ids[:, 1:], top_k=4)
    step = logits.float().abs().max().item() * torch.finfo(dtype).eps / 2
    assert (r.logprob[:, :-1] - ref.logprob).abs().max().item() <= 2 * step + 1e-4
    assert (r.logprob[:, -1] == 0).all() and r.top_ids.shape == (3, 40, 4)
    # half of the prompt, then the rest from its cache; the last row of the first half has the next token as its target
    t1 = ids[:, 1:21].contiguous()
    first, c1 = m.score(ids[:, :20], targets=t1)
    second, _ = m.score(ids[:, 20:], cache=c1)
    whole, _ = m.score(ids)
    both = torch.cat([first.logprob, second.logprob], 1)
    tol = 1e-4 if dtype == F32 else 4 * step + 1e-2
    assert (both - whole.logprob).abs().max().item() <= tol


def test_precision_study_from_recorded_alternatives():
    """The fp32 model's top logits recorded once, then the bf16 model against them: quant_eval's calls in 64 bits."""
    cfg, ref = small_model(MambaLM, F32)
    _, low = small_model(TPMambaLM, BF)
    ids = torch.randint(0, cfg.vocab_size, (2, 30), generator=torch.Generator().manual_seed(2)).to(dev())
    ref_logits, _ = ref.prefill(ids)
    q, _ = low.prefill(ids)
    top_ids, top_lp = quant_eval.record_top_logits(ref_logits, 32)
    xa = f64(ref_logits).reshape(60, -1)
    np.testing.assert_array_equal(top_ids.cpu().numpy().reshape(60, 32), R.top(xa, 32))
    kl = quant_eval.topk_kl(top_ids, top_lp, q)
    qa = f64(q).reshape(60, -1)
    want = R.distill_loss(qa, R.top(xa, 32), f64(top_lp).reshape(60, 32)).reshape(2, 30).mean(1)
    np.testing.assert_allclose(f64(kl), want, atol=1e-5)
    nll = quant_eval.sequence_nll(q, ids)
    lp = R.token_logprob(qa.reshape(2, 30, -1)[:, :-1].reshape(58, -1), ids[:, 1:].cpu().numpy().reshape(58))
    np.testing.assert_allclose(f64(nll), -lp.reshape(2, 29).mean(1), atol=1e-5)


def test_distillation_step_through_the_lm_head():
    """Student logits from a torch product, the distillation gradient carried on to the weight: the one-call form and
    autograd give the same gradient of the weight as the formula in 64 bits."""
    h = make(50, 32, F32, 1, 1.0)
    w = make(400, 32, F32, 2, 0.3).requires_grad_()
    ids, vals = teacher_for((h @ w.detach().T) * 1.5, 12)
    rw = torch.full((50,), 1 / 50, device=dev())
    (P.distill_topk_loss(h @ w.T, ids, vals) * rw).sum().backward()
    one = w.grad.clone()
    w.grad = None
    logits = h @ w.T
    _, grad = P.distill_topk_loss_and_grad(logits.detach(), ids, vals, rw)
    logits.backward(grad)
    x = f64(logits)
    want = R.distill_grad(x, ids.cpu().numpy(), f64(vals), f64(rw))[0].T @ f64(h)
    for got in (one, w.grad):
        np.testing.assert_allclose(f64(got), want, atol=1e-5 * np.abs(want).max())


def test_step_alternatives_in_a_decode_loop():
    """Tokens from the alternatives of each step are those of generate(), whose argmax is the same logits' largest."""
    cfg, m = small_model(TPMambaLM, BF)
    ids = torch.randint(0, cfg.vocab_size, (2, 16), generator=torch.Generator().manual_seed(3)).to(dev())
    want = m.generate(ids, 6)
    logits, cache = m.prefill(ids)
    out = [ids]
    for _ in range(6):
        r = P.token_logprobs(logits[:, -1], top_k=3)
        nxt = r.top_ids[:, :1]
        out.append(nxt)
        logits = m.step(nxt, cache)
    assert torch.equal(torch.cat(out, 1), want)


@pytest.mark.parametrize("temperature", [1e-6, 1e6])
@pytest.mark.parametrize("rows", [3, WARP_ROWS])
def test_extreme_temperatures(temperature, rows):
    """The ends of the allowed range: one token of probability 1, and all nearly equal; masked logits stay out."""
    x = make(rows, 700, F32, 12)
    x[:, 5::7] = float("-inf")
    check_forward(x, targets_for(rows, 700), 9, temperature)
    g = torch.ones(rows, device=dev())
    leaf = x.detach().requires_grad_()
    r = P.token_logprobs(leaf, targets_for(rows, 700), temperature=temperature)
    (grad,) = torch.autograd.grad([r.logprob], [leaf], [g])
    check_grad(x, targets_for(rows, 700), g, torch.zeros_like(g), grad, temperature)


def test_a_backward_pass_on_another_stream_than_the_forward():
    """autograd runs the backward pass on the forward's stream; the caller's stream waits for it."""
    x = make(200, 5001, BF, 13)
    t = targets_for(200, 5001)
    g = torch.ones(200, device=dev())
    leaf = x.detach().requires_grad_()
    (want,) = torch.autograd.grad([P.token_logprobs(leaf, t).logprob], [leaf], [g])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf2 = x.detach().requires_grad_()
        lp = P.token_logprobs(leaf2, t).logprob
    torch.cuda.current_stream().wait_stream(side)
    (got,) = torch.autograd.grad([lp], [leaf2], [g])
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_teacher_values_that_are_no_numbers():
    x = make(3, 90, F32, 14)
    ids = torch.tensor([[1, 2, 3]] * 3, device=dev())
    vals = torch.tensor([[0.0, float("nan"), 1.0], [0.0, float("inf"), 1.0], [0.0, 0.5, 1.0]], device=dev())
    loss, grad = P.distill_topk_loss_and_grad(x, ids, vals, torch.ones(3, device=dev()))
    assert torch.isnan(loss[:2]).all() and torch.isfinite(loss[2])
    assert torch.isnan(grad[:2]).all() and torch.isfinite(grad[2]).all()
