"""Operators on logits: the log probabilities of given tokens with entropy and top
alternatives, the distillation loss from a teacher's top logits, and log probabilities
taken straight from hidden states and the (tied) lm_head matrix.

Logits are [..., V] CUDA tensors (float32, bfloat16 or float16) whose rows may be strided
(``logits[:, :-1]``, a vocabulary whose padding columns are cut off); every statistic and
per-row result is float32.  ``token_logprobs`` and ``distill_topk_loss`` are
differentiable with respect to the logits (reverse mode, once).  Calls run on the current
stream of the logits' device, allocate through torch only and keep nothing, so they can be
captured in a CUDA graph.  (As ever in torch, a captured backward pass wants no graph of an
uncaptured pass over the same leaf alive.)  The reference has no counterpart; the nearest is the
full-vocabulary KL of ``mamba_lite/quant_eval.py:48-68``."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L

__all__ = ["MAX_TOP", "TokenLogprobs", "token_logprobs", "distill_topk_loss", "distill_topk_loss_and_grad",
           "lm_head_logprobs"]

MAX_TOP = 128  # alternatives, or teacher entries, per row
MAX_VOCAB = 1 << 30

_INT_TYPES = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


class TokenLogprobs(NamedTuple):
    """Per row, None where not asked for: the given token's log probability, the entropy of the
    distribution (nats), and the most likely tokens with their log probabilities [..., top_k]."""
    logprob: torch.Tensor | None
    entropy: torch.Tensor | None
    top_ids: torch.Tensor | None
    top_logprobs: torch.Tensor | None


# ------------------------------------------------------------------ arguments
def _refuse_tangent(x: torch.Tensor, what: str) -> None:
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def _check_logits(x: torch.Tensor, what: str) -> None:
    L.require_cuda(x, what)
    L.dtype_code(x.dtype)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{what}: logits need a last dimension of at least one token, got shape {tuple(x.shape)}")
    if x.shape[-1] > MAX_VOCAB:
        raise ValueError(f"{what}: {x.shape[-1]} tokens, at most {MAX_VOCAB}")
    _refuse_tangent(x, what)


def _check_ids(ids: torch.Tensor, shape, device, what: str, name: str) -> torch.Tensor:
    if ids.dtype not in _INT_TYPES:
        raise TypeError(f"{what}: {name} must be integers, got {ids.dtype}")
    if ids.shape != shape:
        raise ValueError(f"{what}: {name} have shape {tuple(ids.shape)}, expected {tuple(shape)}")
    if ids.device != device:
        raise ValueError(f"{what}: {name} are on {ids.device}, the logits on {device}")
    if ids.dtype != torch.int64:
        ids = ids.to(torch.int64)
    return ids if ids.is_contiguous() else ids.contiguous()


def _check_rows(v: torch.Tensor, shape, device, what: str, name: str) -> torch.Tensor:
    if not v.dtype.is_floating_point:
        raise TypeError(f"{what}: {name} must be floating point, got {v.dtype}")
    if v.shape != shape:
        raise ValueError(f"{what}: {name} has shape {tuple(v.shape)}, expected {tuple(shape)}")
    if v.device != device:
        raise ValueError(f"{what}: {name} is on {v.device}, the logits on {device}")
    return v.detach().float().contiguous()


def _check_top_k(top_k: int, vocab: int, what: str) -> int:
    if not 0 <= top_k <= min(MAX_TOP, vocab):
        raise ValueError(f"{what}: top_k = {top_k} must be between 0 and min({vocab} tokens, {MAX_TOP})")
    return int(top_k)


def _check_temperature(t: float, what: str) -> float:
    t = float(t)
    if not 1e-6 <= t <= 1e6:
        raise ValueError(f"{what}: temperature must be between 1e-6 and 1e6, got {t}")
    return t


def _row_layout(x: torch.Tensor):
    """(x, outer, inner, ld_outer, ld) with row (o, i) of x at o * ld_outer + i * ld elements; x is
    copied only if its rows do not lie on two strides or its last dimension is not dense."""
    v = x.shape[-1]
    if x.numel() == 0:
        return x, 0, 0, 0, v
    if x.stride(-1) != 1 and v > 1:
        x = x.contiguous()
    groups: list[list[int]] = []
    for n, st in zip(x.shape[:-1], x.stride()[:-1]):
        if n == 1:
            continue
        if groups and groups[-1][1] == st * n:
            groups[-1] = [groups[-1][0] * n, st]
        else:
            groups.append([n, st])
    if len(groups) > 2:
        x = x.contiguous()
        groups = [[x.numel() // v, v]]
    while len(groups) < 2:
        groups.insert(0, [1, 0])
    (outer, ld_outer), (inner, ld) = groups
    return x, outer, inner, ld_outer, (ld if inner > 1 else v)


def _grad_like(x: torch.Tensor, inner: int, ld_outer: int, ld: int):
    """(gradient of x, its ld_outer, its ld), uninitialised.  The gradient takes x's strides and its
    offset within 16 bytes, so that a row of both has the same alignment and the kernels can use
    16-byte accesses; where x overlaps itself or has large gaps it is contiguous instead."""
    v = x.shape[-1]
    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return torch.empty_like(x), ld_outer, ld
    steps = sorted((st, n) for n, st in zip(x.shape, x.stride()) if n > 1)
    extent = 1 + sum((n - 1) * st for st, n in steps)
    apart = all(st > 0 for st, _ in steps) and all(b >= a * n for (a, n), (b, _) in zip(steps, steps[1:]))
    if not apart or extent > x.numel() + x.numel() // 4 + 4096:
        return torch.empty(x.shape, device=x.device, dtype=x.dtype), inner * v, v
    off = x.data_ptr() % 16 // x.element_size()
    buf = torch.empty(extent + off, device=x.device, dtype=x.dtype)
    return buf.as_strided(x.shape, x.stride(), off), ld_outer, ld


def _call(x: torch.Tensor, name: str, *args, stream: bool = True) -> None:
    """The entry point ``name`` with x's device as the current one, on its current stream."""
    if x.device.index == torch.cuda.current_device():
        L.call(name, *args, *((L.stream_ptr(),) if stream else ()))
    else:
        with torch.cuda.device(x.device):
            L.call(name, *args, *((L.stream_ptr(),) if stream else ()))


def _row_like(x: torch.Tensor, ids: torch.Tensor | None) -> torch.Tensor:
    """An uninitialised fp32 value per row of x; ids [...] or None has x's leading shape."""
    if ids is not None:  # the cheapest of torch's allocating calls
        return torch.empty_like(ids, dtype=torch.float32)
    return x.new_empty(x.shape[:-1], dtype=torch.float32)


def _f32(g: torch.Tensor | None) -> torch.Tensor | None:
    """A row gradient as the kernels read it: dense fp32 (autograd may hand on an expanded scalar)."""
    if g is None or (g.dtype == torch.float32 and g.is_contiguous()):
        return g
    return g.float().contiguous()


# ------------------------------------------------------------------ log probabilities
def _logprobs_fwd(x, targets, top_k, temperature, entropy, want_stats):
    lp = None if targets is None else _row_like(x, targets)
    ent = _row_like(x, targets) if entropy else None
    stats = x.new_empty((*x.shape[:-1], 2), dtype=torch.float32) if want_stats else None
    ids = tlp = None
    if top_k:
        ids = x.new_empty((*x.shape[:-1], top_k), dtype=torch.int64)
        tlp = torch.empty_like(ids, dtype=torch.float32)
    x, outer, inner, ld_outer, ld = _row_layout(x)
    _call(x, "mtp_token_logprobs", x.data_ptr(), L.dtype_code(x.dtype), outer, inner, ld_outer, ld, x.shape[-1],
          L.ptr(targets), temperature, L.ptr(lp), L.ptr(ent), L.ptr(stats), top_k, L.ptr(ids), L.ptr(tlp))
    return lp, ent, stats, ids, tlp


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, targets, top_k, temperature, entropy):
        ctx.set_materialize_grads(False)
        lp, ent, stats, ids, tlp = _logprobs_fwd(x, targets, top_k, temperature, entropy, True)
        ctx.save_for_backward(x, targets, stats, ent)
        ctx.temperature = temperature
        if top_k:
            ctx.mark_non_differentiable(ids, tlp)
        return lp, ent, ids, tlp

    @staticmethod
    @once_differentiable
    def backward(ctx, g, h, *_):
        x, targets, stats, ent = ctx.saved_tensors
        if g is None and h is None:
            return None, None, None, None, None
        return _logprobs_bwd(x, targets, ctx.temperature, stats, ent, g, h), None, None, None, None


def _logprobs_bwd(x, targets, temperature, stats, ent, g, h):
    g, h = _f32(g), _f32(h)
    x, outer, inner, ld_outer, ld = _row_layout(x)
    grad, g_ld_outer, g_ld = _grad_like(x, inner, ld_outer, ld)
    _call(x, "mtp_token_logprobs_bwd", x.data_ptr(), L.dtype_code(x.dtype), outer, inner, ld_outer, ld, x.shape[-1],
          L.ptr(targets), temperature, stats.data_ptr(), L.ptr(ent), L.ptr(g), L.ptr(h), grad.data_ptr(), g_ld_outer, g_ld)
    return grad


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor | None = None, *, top_k: int = 0,
                   temperature: float = 1.0, entropy: bool = True) -> TokenLogprobs:
    """Log probabilities of ``targets`` [...] under softmax(logits [..., V] / temperature), the entropy
    of each row, and its ``top_k`` <= 128 most likely tokens (equal logits: the lower id first).

    A negative target is no token: log probability 0 and no gradient from it (padding).  A target
    >= V gives NaN.  Logits of -inf are tokens of probability 0; a row of nothing else has log
    probabilities -inf, entropy 0 and no gradient.  A NaN or +inf in a row gives NaN.
    ``logprob`` and ``entropy`` are differentiable with respect to the logits, the alternatives
    are not."""
    what = "token_logprobs"
    _check_logits(logits, what)
    if targets is not None:
        targets = _check_ids(targets, logits.shape[:-1], logits.device, what, "targets")
    top_k = _check_top_k(top_k, logits.shape[-1], what)
    temperature = _check_temperature(temperature, what)
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobsFn.apply(logits, targets, top_k, temperature, entropy))
    lp, ent, _, ids, tlp = _logprobs_fwd(logits, targets, top_k, temperature, entropy, False)
    return TokenLogprobs(lp, ent, ids, tlp)


# ------------------------------------------------------------------ distillation
def _teacher(logits, ids, values, what):
    if ids.dim() != logits.dim() or not 1 <= ids.shape[-1] <= MAX_TOP:
        raise ValueError(f"{what}: teacher ids have shape {tuple(ids.shape)}, expected {tuple(logits.shape[:-1])} and "
                         f"1 to {MAX_TOP} entries")
    shape = torch.Size((*logits.shape[:-1], ids.shape[-1]))
    ids = _check_ids(ids, shape, logits.device, what, "teacher ids")
    if values.shape != shape:
        raise ValueError(f"{what}: teacher logits have shape {tuple(values.shape)}, expected {tuple(shape)}")
    if values.device != logits.device:
        raise ValueError(f"{what}: teacher logits are on {values.device}, the logits on {logits.device}")
    L.dtype_code(values.dtype)
    return ids, values.detach().contiguous()


def _distill_fwd(x, ids, values, temperature, want_stats):
    loss = _row_like(x, None)
    stats = x.new_empty((*x.shape[:-1], 2), dtype=torch.float32) if want_stats else None
    x, outer, inner, ld_outer, ld = _row_layout(x)
    _call(x, "mtp_distill_topk", x.data_ptr(), L.dtype_code(x.dtype), outer, inner, ld_outer, ld, x.shape[-1],
          ids.data_ptr(), values.data_ptr(), L.dtype_code(values.dtype), ids.shape[-1], temperature, loss.data_ptr(),
          L.ptr(stats))
    return loss, stats


def _distill_grad(x, ids, values, temperature, stats, weight, want_loss):
    loss = _row_like(x, None) if want_loss else None
    x, outer, inner, ld_outer, ld = _row_layout(x)
    grad, g_ld_outer, g_ld = _grad_like(x, inner, ld_outer, ld)
    _call(x, "mtp_distill_topk_grad", x.data_ptr(), L.dtype_code(x.dtype), outer, inner, ld_outer, ld, x.shape[-1],
          ids.data_ptr(), values.data_ptr(), L.dtype_code(values.dtype), ids.shape[-1], temperature, L.ptr(stats),
          weight.data_ptr(), L.ptr(loss), grad.data_ptr(), g_ld_outer, g_ld)
    return loss, grad


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, values, temperature):
        loss, stats = _distill_fwd(x, ids, values, temperature, True)
        ctx.save_for_backward(x, ids, values, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, ids, values, stats = ctx.saved_tensors
        _, grad = _distill_grad(x, ids, values, ctx.temperature, stats, _f32(g), False)
        return grad, None, None, None


def distill_topk_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *,
                      temperature: float = 1.0) -> torch.Tensor:
    """KL(q || p) per row [...] of p = softmax(logits / temperature) from the teacher's distribution over
    its k <= 128 recorded tokens, q = softmax(teacher_logits [..., k] / temperature) at
    ``teacher_ids`` [..., k].  ``teacher_logits`` may be log probabilities (``token_logprobs``'s
    alternatives): q is the same.

    An entry with a negative id or a logit of -inf is not used; a row without a used entry has loss
    0 and no gradient; a used id >= V gives NaN; equal ids add up.  Differentiable with respect
    to ``logits`` only.  Not scaled by temperature squared."""
    what = "distill_topk_loss"
    _check_logits(logits, what)
    ids, values = _teacher(logits, teacher_ids, teacher_logits, what)
    temperature = _check_temperature(temperature, what)
    if logits.requires_grad and torch.is_grad_enabled():
        return _DistillFn.apply(logits, ids, values, temperature)
    return _distill_fwd(logits, ids, values, temperature, False)[0]


@torch.no_grad()
def distill_topk_loss_and_grad(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                               row_weight: torch.Tensor, *, temperature: float = 1.0):
    """``distill_topk_loss`` and the gradient of ``(row_weight * loss).sum()`` with respect to the logits
    (in their dtype) in one call: the logits are read from memory once instead of once for each
    pass.  Rows of weight 0 have gradient 0.  Outside autograd: feed the gradient on with
    ``logits.backward(grad)``."""
    what = "distill_topk_loss_and_grad"
    _check_logits(logits, what)
    ids, values = _teacher(logits, teacher_ids, teacher_logits, what)
    weight = _check_rows(row_weight, logits.shape[:-1], logits.device, what, "row_weight")
    return _distill_grad(logits, ids, values, _check_temperature(temperature, what), None, weight, True)


# ------------------------------------------------------------------ from hidden states
def lm_head_logprobs(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor | None = None, *, top_k: int = 0,
                     temperature: float = 1.0, entropy: bool = True) -> TokenLogprobs:
    """``token_logprobs`` of the logits hidden [..., K] @ weight [V, K]^T, accumulated in fp32 and never
    held as a whole: [rows, V] is neither rounded to the model's dtype nor written.  float32 or
    bfloat16, both of one dtype.  No gradient: call it under ``torch.no_grad()``.

    bfloat16 on 16-byte boundaries takes one tensor-core pass without ``top_k``.  With it (and
    otherwise) the logits go through blocks of about 256 MB in fp32, of which the tensor core sums K as
    a whole, truncating (a logit is up to 8.6e-10 K of itself too small), where the pass sums at most
    1024 at a time: for wider models the two differ in the last digits."""
    what = "lm_head_logprobs"
    L.require_cuda(hidden, what)
    if hidden.dtype not in (torch.float32, torch.bfloat16) or weight.dtype != hidden.dtype:
        raise TypeError(f"{what}: hidden and weight must both be float32 or bfloat16, got {hidden.dtype}, {weight.dtype}")
    if hidden.dim() == 0 or weight.dim() != 2 or weight.shape[0] == 0 or hidden.shape[-1] != weight.shape[1] or \
            weight.shape[1] == 0:
        raise ValueError(f"{what}: hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} do not fit")
    if weight.device != hidden.device:
        raise ValueError(f"{what}: weight is on {weight.device}, hidden on {hidden.device}")
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        raise RuntimeError(f"{what} has no gradient; call it under torch.no_grad()")
    _refuse_tangent(hidden, what)
    _refuse_tangent(weight, what)
    lead, (v, k) = hidden.shape[:-1], weight.shape
    if targets is not None:
        targets = _check_ids(targets, lead, hidden.device, what, "targets")
    top_k = _check_top_k(top_k, v, what)
    temperature = _check_temperature(temperature, what)
    x = hidden.reshape(-1, k)
    if max(x.shape[0], v, k) > MAX_VOCAB:
        raise ValueError(f"{what}: {x.shape[0]} rows, {v} tokens or width {k}: at most {MAX_VOCAB}")
    if x.stride(-1) != 1 or not k <= x.stride(0) <= MAX_VOCAB:
        x = x.contiguous()
    if weight.stride(1) != 1 or not k <= weight.stride(0) <= MAX_VOCAB:
        weight = weight.contiguous()
    rows = x.shape[0]
    args = (L.ptr(x), x.stride(0) if rows > 1 else k, rows, k, L.ptr(weight), weight.stride(0) if v > 1 else k, v,
            L.dtype_code(x.dtype))
    lp = None if targets is None else _row_like(hidden, targets)
    ent = _row_like(hidden, targets) if entropy else None
    ids = tlp = None
    if top_k:
        ids = x.new_empty((*lead, top_k), dtype=torch.int64)
        tlp = torch.empty_like(ids, dtype=torch.float32)
    need = C.c_int64(0)
    _call(x, "mtp_lm_head_logprobs_workspace", *args, top_k, C.byref(need), stream=False)
    work = x.new_empty(need.value, dtype=torch.uint8)
    _call(x, "mtp_lm_head_logprobs", *args, L.ptr(targets), temperature, L.ptr(lp), L.ptr(ent), top_k, L.ptr(ids),
          L.ptr(tlp), work.data_ptr(), need.value)
    return TokenLogprobs(lp, ent, ids, tlp)
