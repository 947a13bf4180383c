"""Accuracy metrics of the precision study, with the definitions of
``mamba_lite/quant_eval.py:48-68``: for logits ``ref`` and ``q`` of shape [b, l, V],
per sequence (mean over positions) the KL divergence KL(softmax(ref) || softmax(q)),
the top-1 agreement and the top-5 agreement in order and as a set.  ``summarize``
reduces per-sequence values to mean and standard deviation.

``record_top_logits`` / ``topk_kl`` are the same study from a recorded reference: k tokens a
position instead of the reference's [b, l, V] logits.  ``sequence_nll`` is the mean negative log
likelihood of a sequence's own tokens.  These three run in the kernels of ``logprobs.py``."""
from __future__ import annotations

import torch
import torch.nn.functional as F

from .logprobs import distill_topk_loss, token_logprobs


def quant_metrics(ref: torch.Tensor, q: torch.Tensor) -> dict:
    log_p = F.log_softmax(ref.float(), dim=-1)
    log_q = F.log_softmax(q.float(), dim=-1)
    # sum_v p_v (log p_v - log q_v), per position
    kl_pos = F.kl_div(log_q, log_p, reduction="none", log_target=True).sum(-1)
    top_ref = torch.topk(ref, 5, dim=-1).indices
    top_q = torch.topk(q, 5, dim=-1).indices
    same_set = torch.sort(top_ref, dim=-1).values == torch.sort(top_q, dim=-1).values
    return {
        "kl": kl_pos.mean(dim=1),
        "top1": (top_ref[..., 0] == top_q[..., 0]).float().mean(dim=1),
        "top5_ordered": torch.all(top_ref == top_q, dim=-1).float().mean(dim=1),
        "top5_unordered": torch.all(same_set, dim=-1).float().mean(dim=1),
    }


@torch.no_grad()
def record_top_logits(ref: torch.Tensor, k: int = 64):
    """The k <= 128 most likely tokens of every position of ref [b, l, V]: (ids [b, l, k] int64, log
    probabilities [b, l, k] float32), what ``topk_kl`` needs of the reference model."""
    top = token_logprobs(ref, top_k=k, entropy=False)
    return top.top_ids, top.top_logprobs


@torch.no_grad()
def topk_kl(ids: torch.Tensor, logprobs: torch.Tensor, q: torch.Tensor) -> torch.Tensor:
    """Per sequence (mean over positions) KL of q [b, l, V] from the recorded reference, whose distribution
    is renormalised over its k tokens."""
    return distill_topk_loss(q, ids, logprobs).mean(dim=1)


@torch.no_grad()
def sequence_nll(logits: torch.Tensor, input_ids: torch.Tensor) -> torch.Tensor:
    """Per sequence mean negative log likelihood of input_ids [b, l] under logits [b, l, V] (position i
    predicts token i + 1; negative ids are padding and do not count); exp of it is the perplexity.  A
    sequence with no token to predict has 0."""
    targets = input_ids[:, 1:]
    logprob = token_logprobs(logits[:, :-1], targets, entropy=False).logprob
    return -logprob.sum(dim=1) / (targets >= 0).sum(dim=1).clamp(min=1)


def summarize(per_sequence: dict) -> dict:
    out = {}
    for name, values in per_sequence.items():
        v = torch.as_tensor(values, dtype=torch.float64).flatten()
        out[name] = {"mean": float(v.mean()), "std": float(v.std()) if v.numel() > 1 else 0.0}
    return out
