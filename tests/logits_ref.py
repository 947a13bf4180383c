"""The operators of logprobs.py in 64-bit numpy, from their definitions, and the error bounds the GPU tests hold
the kernels to.

Bounds.  u = 2^-24 is the relative rounding error of an fp32 operation.  A row's sums run over at most V / 256 + 64
terms in a chain (one thread's elements, then the joins), each addition off by u of the running sum, and each
term e^d by at most 2^-22 (the hardware exponential) + 2 u |d| (its argument), where the sum over terms of
e^d |d| is at most (log S + 1) S.  So S is known to a relative B = (V / 256 + 64) u + 2^-22 + 2 u (log S + 1), and
log S to B plus two roundings.  Every derived value below adds the roundings of its own last steps."""
import numpy as np

U = 2.0 ** -24


def softmax_parts(x, temperature):
    """x [rows, V] -> (z, m, log S) in 64 bits, z = x / temperature; rows of -inf alone have m = -inf."""
    z = np.asarray(x, np.float64) / temperature
    with np.errstate(invalid="ignore"):
        m = z.max(-1, keepdims=True)
        d = np.where(np.isneginf(m), -np.inf, z - m)
        log_s = np.log(np.where(np.isneginf(m), 1.0, np.exp(d).sum(-1, keepdims=True)))
    return z, m, log_s, d


def log_probs(x, temperature=1.0):
    _, _, log_s, d = softmax_parts(x, temperature)
    with np.errstate(invalid="ignore"):
        return d - log_s


def entropy(x, temperature=1.0):
    lp = log_probs(x, temperature)
    with np.errstate(invalid="ignore"):
        p = np.exp(lp)
        return -np.where(p == 0, 0.0, p * lp).sum(-1)


def token_logprob(x, targets, temperature=1.0):
    v = x.shape[-1]
    lp = log_probs(x, temperature)
    out = np.take_along_axis(lp, np.clip(targets, 0, v - 1)[:, None], 1)[:, 0]
    out = np.where(targets >= v, np.nan, out)
    return np.where(targets < 0, 0.0, out)


def top(x, k):
    """Indices of the k largest: NaN first, then falling, the lower index first among equals."""
    x = np.asarray(x, np.float64)
    key = np.where(np.isnan(x), np.inf, x)
    order = np.lexsort((np.broadcast_to(np.arange(x.shape[-1]), x.shape), -key, ~np.isnan(x)), axis=-1)
    return order[:, :k]


def token_logprobs_grad(x, targets, g, h, temperature=1.0):
    """Gradient of sum g logprob + h entropy; also the sum of the magnitudes of its terms."""
    v = x.shape[-1]
    lp = log_probs(x, temperature)
    p = np.exp(lp)
    ent = entropy(x, temperature)[:, None]
    g = np.where(targets < 0, 0.0, np.asarray(g, np.float64))[:, None]
    h = np.asarray(h, np.float64)[:, None]
    lpc = np.where(p == 0, 0.0, lp)
    onehot = (np.arange(v)[None, :] == targets[:, None]).astype(np.float64)
    empty = np.isneginf(lp).all(-1, keepdims=True)
    grad = (g * (onehot - p) - h * p * (lpc + ent)) / temperature
    mag = (np.abs(g) * (onehot + p) + np.abs(h) * p * (np.abs(lpc) + np.abs(ent) + 1)) / temperature
    return np.where(empty, 0.0, grad), mag


def teacher(ids, values, temperature=1.0):
    used = (ids >= 0) & ~np.isneginf(values)
    t = np.where(used, np.asarray(values, np.float64) / temperature, -np.inf)
    any_used = used.any(-1, keepdims=True)
    m = np.where(any_used, t.max(-1, keepdims=True), 0.0)
    with np.errstate(divide="ignore", invalid="ignore"):
        log_q = np.where(any_used, t - m - np.log(np.exp(t - m).sum(-1, keepdims=True)), -np.inf)
    return np.exp(log_q), log_q


def distill_loss(x, ids, values, temperature=1.0):
    v = x.shape[-1]
    q, log_q = teacher(ids, values, temperature)
    lp = np.take_along_axis(log_probs(x, temperature), np.clip(ids, 0, v - 1), 1)
    lp = np.where((ids >= v) & (q > 0), np.nan, lp)
    with np.errstate(invalid="ignore"):
        return np.where(q > 0, q * (log_q - lp), 0.0).sum(-1)


def distill_grad(x, ids, values, w, temperature=1.0):
    q, _ = teacher(ids, values, temperature)
    lp = log_probs(x, temperature)
    p = np.exp(lp)
    target = np.zeros_like(p)
    for r in range(x.shape[0]):
        for j, qq in zip(ids[r], q[r]):
            if qq > 0:
                target[r, j] += qq
    w = np.asarray(w, np.float64)[:, None] / temperature
    empty = np.isneginf(lp).all(-1, keepdims=True) | (q.sum(-1, keepdims=True) == 0)
    return np.where(empty, 0.0, w * (p - target)), np.abs(w) * (p + target)


# ------------------------------------------------------------------ bounds
def sum_bound(x, temperature=1.0):
    """Relative error bound B of a row's S [rows]."""
    log_s = softmax_parts(x, temperature)[2][:, 0]
    return (x.shape[-1] / 256 + 64) * U + 2.0 ** -22 + 2 * U * (log_s + 1)


def logprob_bound(x, lp, temperature=1.0):
    """Of a log probability lp [rows, ...]: B, and four roundings of values no larger than |lp| + 2 log S."""
    b = sum_bound(x, temperature)
    log_s = softmax_parts(x, temperature)[2][:, 0]
    shape = (-1,) + (1,) * (np.ndim(lp) - 1)
    return b.reshape(shape) + 4 * U * (np.abs(np.where(np.isfinite(lp), lp, 0)) + 2 * log_s.reshape(shape) + 1)


def entropy_bound(x, temperature=1.0):
    """log S - Q / S with Q = sum e^d d: both sums to B, |Q / S| = log S - H."""
    _, _, log_s, _ = softmax_parts(x, temperature)
    log_s = log_s[:, 0]
    ent = entropy(x, temperature)
    ent = np.where(np.isfinite(ent), ent, 0)
    return sum_bound(x, temperature) * (1 + 3 * (np.abs(log_s - ent) + 1)) + 4 * U * (log_s + 1)


def grad_bound(x, grad, mag, eps, tiny, temperature=1.0):
    """The terms of a gradient (magnitudes mag) to B, the exponential's error and four roundings, the entropy's error
    in its factor (mag holds |h| p + ...), then half a step of the gradient's own type."""
    b = sum_bound(x, temperature)[:, None]
    lp = log_probs(x, temperature)
    lp = np.where(np.isfinite(lp), np.abs(lp), 0)
    # an exponential whose argument is lp (|lp| <= 110 where it does not vanish): relative 2 u |lp| + 2^-22
    rel = b + 2.0 ** -22 + 4 * U * (np.minimum(lp, 110) + 2) + entropy_bound(x, temperature)[:, None]
    return mag * rel + np.abs(grad) * eps / 2 + tiny


# ------------------------------------------------------------------ hidden states whose products add up exactly
SUM_GRAIN, SUM_LIMIT = 2.0 ** -11, 2.0 ** 13  # every sum of up to 1024 products is a multiple of one below the other


def exact_score_inputs(rows, v, k, seed=0):
    """(hidden [rows, K], weight [V, K]) in bf16 values, products of which add up without rounding in 24 bits over any 1024
    (any order) but not over more.  Of 16 positions 15 give 8.5, 960 of them 8160; one gives an odd multiple of 2^-11 for
    an even token and an even one for an odd token, 64 of them less than 4.  A sum that goes past 2^13 in 24 bits loses an
    odd multiple's last bit at every step and an even multiple's never, so that the tokens drift apart."""
    g = np.random.default_rng(seed)
    h, w = np.ones((rows, k)), np.full((v, k), 8.5)
    fine = np.arange(k) % 16 == 7
    h[:, fine] = np.where(g.random((rows, fine.sum())) < 0.5, -1, 1) * 2.0 ** -5
    w[:, fine] = (2 * g.integers(0, 63, (v, fine.sum())) + (np.arange(v) % 2 == 0)[:, None]) * 2.0 ** -6
    return h, w


def score_accumulators(k):
    """Positions that one accumulator sums: 64-wide blocks of K in equal numbers, 16 blocks at most."""
    blocks = -(-k // 64)
    splits = -(-blocks // 16)
    return 64 * -(-blocks // splits)


def exact_score_bounds(h, w, targets, per_acc=None):
    """(logits, logprob, its bound, entropy, its bound).  The accumulators (per_acc positions each) are exact; each is
    added to the ones before it with one rounding, half a step of the sum.  dz is the sum of those.  A log
    probability moves by at most 2 dz, an entropy by dz sum p |log p + H| to first order, of which 2 dz covers the rest
    (dz < 2^-8)."""
    x = h @ w.T
    dz = np.zeros(len(h))
    if per_acc:
        for end in range(2 * per_acc, w.shape[1] + per_acc, per_acc):
            part = np.abs(h[:, :end] @ w[:, :end].T).max(-1)
            dz += 2.0 ** np.floor(np.log2(part)) * U
    lp, ent = log_probs(x), entropy(x)
    want = token_logprob(x, targets)
    drift = (np.exp(lp) * np.abs(lp + ent[:, None])).sum(-1)
    return x, want, logprob_bound(x, want) + 2 * dz, ent, entropy_bound(x) + 2 * dz * drift
