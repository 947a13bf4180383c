"""Operators on logits at the ends of their ranges, against the 64-bit definitions with the bounds of logits_ref.py."""
import pytest
import torch

from mamba_tp_lite_b200 import logprobs as P
from tests.gpu_util import dev
from tests.test_gpu_logprobs import BF, F16, F32, check_distill, check_forward, check_grad, make, targets_for, teacher_for

pytestmark = pytest.mark.gpu


def test_a_used_teacher_entry_past_the_vocabulary_is_reported_however_unlikely():
    """exp(-200) is 0 in fp32, but the entry is used: its id counts, not its probability."""
    v = 90
    x = make(4, v, F32, 15)
    ids = torch.tensor([[1, v], [1, 2], [v, 1], [v, 1]], device=dev())
    vals = torch.tensor([[0.0, -200.0], [0.0, -200.0], [float("-inf"), 0.0], [torch.finfo(F32).min, 0.0]], device=dev())
    w = torch.ones(4, device=dev())
    for loss, grad in (P.distill_topk_loss_and_grad(x, ids, vals, w), (P.distill_topk_loss(x, ids, vals), None)):
        assert torch.isnan(loss).tolist() == [True, False, False, True]
        if grad is not None:
            assert torch.isnan(grad).all(1).tolist() == [True, False, False, True]
            assert torch.isfinite(grad[1:3]).all()


SCALES = [2.0 ** -115, 2.0 ** -100, 2.0 ** -60, 2.0 ** -31, 2.0 ** -29, 2.0 ** 60]


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,v", [(5, 257), (2500, 130)])
def test_gradients_of_small_and_large_upstream_gradients(scale, dtype, rows, v):
    """The gradient is as good relative to a small factor as to a large one."""
    x = make(rows, v, dtype, 16)
    t = targets_for(rows, v)
    g = torch.linspace(0.5, 1.5, rows, device=dev()) * scale
    h = torch.linspace(-1, 0.9, rows, device=dev()) * scale
    zero = torch.zeros_like(g)
    for gg, hh in ((g, h), (g, zero), (zero, h), (g, h / scale), (g / scale, h)):
        leaf = x.detach().requires_grad_()
        r = P.token_logprobs(leaf, t)
        outs = [(r.logprob, gg)] + ([] if hh is zero else [(r.entropy, hh)])
        (grad,) = torch.autograd.grad([o for o, _ in outs], [leaf], [u for _, u in outs])
        check_grad(x, t, gg, hh, grad)
    ids, vals = teacher_for(x, 20)
    loss, grad = P.distill_topk_loss_and_grad(x, ids, vals, g)
    check_distill(x, ids, vals, g, loss, grad)
    leaf = x.detach().requires_grad_()
    (grad,) = torch.autograd.grad([P.distill_topk_loss(leaf, ids, vals)], [leaf], [g])
    check_distill(x, ids, vals, g, loss, grad)


@pytest.mark.parametrize("rows", [3, 2500])
def test_a_teacher_token_that_the_student_all_but_excludes(rows):
    """q = e^-87 against p = e^-90, below the smallest normal number, under a large weight: p is a twentieth of q."""
    x = torch.full((rows, 80), -80.0, device=dev())
    x[:, 5], x[:, 7] = -90.0, 0.0
    ids = torch.tensor([7, 5], device=dev()).expand(rows, 2)
    vals = torch.tensor([0.0, -87.0], device=dev()).expand(rows, 2)
    w = torch.linspace(0.5, 1.5, rows, device=dev()) * 2.0 ** 100
    loss, grad = P.distill_topk_loss_and_grad(x, ids, vals, w)
    check_distill(x, ids, vals, w, loss, grad)
    leaf = x.detach().requires_grad_()
    (grad,) = torch.autograd.grad([P.distill_topk_loss(leaf, ids, vals)], [leaf], [w])
    check_distill(x, ids, vals, w, loss, grad)


@pytest.mark.parametrize("rows,v", [(6, 50281), (3, 3001), (2500, 1000), (2500, 3001)])
@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("which", ["few", "from_the_middle", "up_to_the_middle", "one_lane"])
def test_masked_logits_that_begin_anywhere_in_a_row(rows, v, dtype, which):
    """The threads of a warp meet their first masked logit at different times, or never."""
    x = make(rows, v, dtype, 17)
    j = torch.arange(v, device=dev())
    banned = {"few": j % 997 == 5, "from_the_middle": j > v // 2, "up_to_the_middle": j < v // 2,
              "one_lane": (j // 8) % 32 == 3}[which]
    x[:, banned] = float("-inf")
    t = targets_for(rows, v)
    for k in (0, 5):
        check_forward(x, t, k)


@pytest.mark.parametrize("rows,v", [(300, 50281), (2500, 1003)])
def test_masked_rows_give_the_same_bits_every_time(rows, v):
    x = make(rows, v, BF, 18)
    x[torch.rand(rows, v, generator=torch.Generator().manual_seed(1)).to(dev()) < 0.003] = float("-inf")
    t = targets_for(rows, v)
    want = P.token_logprobs(x, t, top_k=4)
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(P.token_logprobs(x, t, top_k=4), want))
