"""Operators on logits at the ends of their ranges, against the 64-bit definitions with the bounds of logits_ref.py."""
import pytest
import torch

from mamba_tp_lite_b200 import logprobs as P
from tests.gpu_util import dev
from tests.test_gpu_logprobs import F32, make

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
