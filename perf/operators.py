"""The framework's operators on logits, as they are timed: the log probabilities of given tokens with entropy and top
alternatives (forward, and backward to the logits), the distillation loss from a teacher's top logits (forward, and
forward with gradient), and log probabilities taken straight from hidden states and the lm_head matrix.

``listed()`` gives the cases, ``prepare(case, seed)`` a program's inputs on the GPU, ``run(state)`` one pass: the plain
form in 32-bit torch operations, or with ``own`` set the calls into ``mamba_tp_lite_b200``.  ``exact(case, seed)`` is the
same from the definitions in 64 bits, ``work(case)`` the bytes and operations one pass cannot do without.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}

VOCAB = 50280  # every benchmark shape of the repository


def listed():
    return [
        # one decode step of a single sequence that reports its token's log probability and five alternatives
        dict(name="step_b1", op="logprobs", batch=1, seq=1, vocab=VOCAB, pad=0, dtype="bf16", top_k=5,
             temperature=1.0, masked=False),
        # the same for the decode batch of the benchmark, twenty alternatives
        dict(name="step_b32", op="logprobs", batch=32, seq=1, vocab=VOCAB, pad=0, dtype="bf16", top_k=20,
             temperature=1.0, masked=False),
        # perplexity of the benchmark's prompts from their prefill logits (next tokens: the last position is cut off)
        dict(name="prompt_32x1024", op="logprobs", batch=32, seq=1024, vocab=VOCAB, pad=0, dtype="bf16", top_k=0,
             temperature=1.0, masked=False),
        # recording the fp32 model's top logits for the accuracy study (2 x 1024 tokens)
        dict(name="record_top64", op="logprobs", batch=2, seq=1025, vocab=VOCAB, pad=0, dtype="f32", top_k=64,
             temperature=1.0, masked=False),
        # a ragged batch: a vocabulary whose padding columns are cut off, banned tokens, a sampling temperature
        dict(name="ragged_f16", op="logprobs", batch=3, seq=260, vocab=50277, pad=3, dtype="f16", top_k=7,
             temperature=0.7, masked=True),
        # a training step's log probabilities with an entropy bonus, forward and backward
        dict(name="train_8x1024", op="logprobs_grad", batch=8, seq=1024, vocab=VOCAB, pad=0, dtype="bf16",
             temperature=1.0, masked=False),
        # the same in fp32 on a small odd vocabulary
        dict(name="train_small", op="logprobs_grad", batch=5, seq=27, vocab=1001, pad=0, dtype="f32",
             temperature=1.3, masked=True),
        # the accuracy study against recorded top logits: loss only
        dict(name="distill_eval", op="distill", batch=2, seq=1024, vocab=VOCAB, pad=0, dtype="f32", top_k=64,
             temperature=1.0, grad="none"),
        # a distillation step: the loss and its gradient in one call
        dict(name="distill_8x1024", op="distill", batch=8, seq=1024, vocab=VOCAB, pad=0, dtype="bf16", top_k=64,
             temperature=1.0, grad="joint"),
        # a small softened distillation through autograd
        dict(name="distill_small", op="distill", batch=3, seq=111, vocab=8191, pad=0, dtype="f16", top_k=16,
             temperature=2.0, grad="autograd"),
        # scoring prompts with the 1.4b shape's lm_head, no logits in memory
        dict(name="score_8x1024", op="score", batch=8, seq=1024, vocab=VOCAB, hidden=2048, temperature=1.0),
        # a short prompt on the 130m shape
        dict(name="score_64", op="score", batch=1, seq=64, vocab=VOCAB, hidden=768, temperature=1.0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "logprobs_grad", "distill", "score"])
    batch = _log_uniform(rng, 1, 32)
    if op == "score":
        hidden = 8 * _log_uniform(rng, 32, 320)
        vocab = _log_uniform(rng, 1000, 65536)
        seq = _log_uniform(rng, 1, max(1, min(1024, int(4e8 / (vocab * batch)))))
        return dict(op=op, batch=batch, seq=seq, vocab=vocab, hidden=hidden, temperature=rng.choice([1.0, 1.0, 0.8]))
    vocab = _log_uniform(rng, 1000, 131072)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    most = 4e8 if op == "logprobs" else 2e8
    seq = _log_uniform(rng, 1, max(1, min(1024, int(most / (vocab * batch)))))
    case = dict(op=op, batch=batch, seq=seq, vocab=vocab, pad=rng.choice([0, 0, 1, 5, 8]), dtype=dtype,
                temperature=rng.choice([1.0, 1.0, 0.6, 2.0]))
    if op == "logprobs":
        case.update(top_k=rng.choice([0, 0, 1, 5, 20, 64, 128]), masked=rng.random() < 0.3)
    elif op == "logprobs_grad":
        case.update(masked=rng.random() < 0.3)
    else:
        case.update(top_k=_log_uniform(rng, 1, 128), grad=rng.choice(["none", "joint", "autograd"]))
    return case


# ------------------------------------------------------------------ inputs
def _rows(case):
    """Rows one pass works on: prompt scoring from logits cuts off the last position."""
    cut = 1 if case["op"] == "logprobs" and case["seq"] > 1 else 0
    return case["batch"] * (case["seq"] - cut)


def _logits(case, gen):
    """Language-model-like logits [batch, seq, vocab + pad]: a unigram bias, noise, and a few likely tokens a row."""
    b, l, v = case["batch"], case["seq"], case["vocab"] + case["pad"]
    rows = b * l
    bias = torch.randn(v, generator=gen, device="cuda") * 1.5 - 4.0
    likely = torch.randint(0, case["vocab"], (rows, 8), generator=gen, device="cuda")
    lift = torch.rand(rows, 8, generator=gen, device="cuda") * 8.0 + 2.0
    out = torch.empty(rows, v, device="cuda", dtype=_DTYPES[case["dtype"]])
    for r0 in range(0, rows, 4096):
        blk = torch.randn(min(4096, rows - r0), v, generator=gen, device="cuda")
        blk.mul_(2.0).add_(bias)
        blk.scatter_add_(1, likely[r0:r0 + 4096], lift[r0:r0 + 4096])
        out[r0:r0 + 4096] = blk
    if case.get("masked"):
        banned = _banned(case, gen)
        out[:, :case["vocab"]].masked_fill_(banned, float("-inf"))
    return out.view(b, l, v), likely.view(b, l, 8)


def _banned(case, gen):
    """Tokens no row may take: a tenth of the vocabulary, its first among them, never its last."""
    banned = torch.rand(case["vocab"], generator=gen, device="cuda") < 0.1
    banned[0], banned[-1] = True, False
    return banned


def _targets(case, likely, gen):
    b, l = likely.shape[:2]
    pick = likely.gather(2, torch.randint(0, 8, (b, l, 1), generator=gen, device="cuda"))[..., 0]
    other = torch.randint(0, case["vocab"], (b, l), generator=gen, device="cuda")
    tgt = torch.where(torch.rand(b, l, generator=gen, device="cuda") < 0.7, pick, other)
    if l > 8:  # a padded batch: the end of every other sequence is no token
        cut = l - l // 8
        tgt[1::2, cut:] = -1
    return tgt


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case=case)
    b, l, v, t = case["batch"], case["seq"], case["vocab"], case["temperature"]
    if case["op"] == "score":
        h = case["hidden"]
        st["hidden"] = torch.randn(b, l, h, generator=gen, device="cuda").to(torch.bfloat16)
        st["weight"] = (torch.randn(v, h, generator=gen, device="cuda") * (2.0 / math.sqrt(h))).to(torch.bfloat16)
        likely = torch.randint(0, v, (b, l, 8), generator=gen, device="cuda")
        st["targets"] = _targets(case, likely, gen)
        return st
    x, likely = _logits(case, gen)
    if case["op"] == "distill":
        # the teacher: the student's logits with noise on them, its top logits as recorded (fp32 values)
        k = case["top_k"]
        st["ids"] = torch.empty(b * l, k, device="cuda", dtype=torch.int64)
        st["values"] = torch.empty(b * l, k, device="cuda", dtype=torch.float32)
        flat = x.view(b * l, -1)[:, :v]
        for r0 in range(0, b * l, 2048):
            blk = flat[r0:r0 + 2048].float()
            blk = blk + torch.randn(blk.shape, generator=gen, device="cuda") * 0.7
            top = blk.topk(k, dim=-1)
            st["ids"][r0:r0 + 2048] = top.indices
            st["values"][r0:r0 + 2048] = top.values
        st["ids"] = st["ids"].view(b, l, k)
        st["values"] = st["values"].view(b, l, k)
        st["logits"] = x[..., :v]
        w = torch.rand(b, l, generator=gen, device="cuda") + 0.5
        if l > 8:
            w[1::2, l - l // 8:] = 0.0  # padded positions carry no weight
        st["weight"] = w / _mean(case)
        return st
    tgt = _targets(case, likely, gen)
    if case.get("masked"):  # a given token is one the row may take
        last = x[..., :v].gather(2, tgt.clamp(min=0).unsqueeze(-1))[..., 0]
        tgt = torch.where((last == float("-inf")) & (tgt >= 0), torch.full_like(tgt, v - 1), tgt)
    st["logits"] = x[..., :v]
    if case["op"] == "logprobs" and l > 1:
        st["logits"], tgt = x[:, :-1, :v], tgt[:, 1:].contiguous()
    st["targets"] = tgt
    if case["op"] == "logprobs_grad":
        st["d_logprob"] = -torch.rand(b, l, generator=gen, device="cuda") / _mean(case)
        st["d_entropy"] = torch.full((b, l), -0.01 / _mean(case), device="cuda")
    return st


def _mean(case):
    """A loss is a mean over the rows; with fp16 logits the program scales it up so that gradients stay normal."""
    return 1.0 if case["dtype"] == "f16" else case["batch"] * case["seq"]


# ------------------------------------------------------------------ the plain form (32 bits)
def _plain_softmax(z):
    """(z - max, log of the sum of e^(z - max)) over the last dimension."""
    d = z - z.amax(-1, keepdim=True)
    return d, d.exp().sum(-1, keepdim=True).log()


def _plain_logprob(d, log_s, targets):
    safe = targets.clamp(min=0).unsqueeze(-1)
    lp = (d.gather(-1, safe) - log_s).squeeze(-1)
    return torch.where(targets >= 0, lp, torch.zeros_like(lp))


def _plain_entropy(d, log_s):
    lp = d - log_s
    return -torch.where(lp > float("-inf"), lp.exp() * lp, torch.zeros_like(lp)).sum(-1)


def _plain_top(x, k):
    """Indices of the k largest of the last dimension, ties to the lowest index: one integer key per element."""
    bits = (x.float() + 0.0).view(torch.int32)
    order = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).to(torch.int64)
    n = x.shape[-1]
    key = order * (1 << 32) + torch.arange(n - 1, -1, -1, device=x.device)
    return n - 1 - (key.topk(k, dim=-1).values & 0xFFFFFFFF)


def _run_plain(st):
    case = st["case"]
    temp = case["temperature"]
    if case["op"] == "score":
        z = (st["hidden"].float() @ st["weight"].float().T) / temp
        d, log_s = _plain_softmax(z)
        return {"logprob": _plain_logprob(d, log_s, st["targets"]), "entropy": _plain_entropy(d, log_s)}
    x = st["logits"]
    d, log_s = _plain_softmax(x.float() / temp)
    if case["op"] == "distill":
        q, log_q = _plain_teacher(st)
        log_p = d.gather(-1, st["ids"]) - log_s
        loss = torch.where(q > 0, q * (log_q - log_p), torch.zeros_like(q)).sum(-1)
        if case["grad"] == "none":
            return {"loss": loss}
        grad = (d - log_s).exp()
        grad.scatter_add_(-1, st["ids"], -q)
        grad.mul_((st["weight"] / temp).unsqueeze(-1))
        return {"loss": loss, "grad": grad.to(x.dtype)}
    out = {"logprob": _plain_logprob(d, log_s, st["targets"]), "entropy": _plain_entropy(d, log_s)}
    if case["op"] == "logprobs":
        if case["top_k"]:
            ids = _plain_top(x, case["top_k"])
            out["top_ids"] = ids
            out["top_logprobs"] = d.gather(-1, ids) - log_s
        return out
    lp = d - log_s
    p = lp.exp()
    g = torch.where(st["targets"] >= 0, st["d_logprob"], torch.zeros_like(st["d_logprob"])).unsqueeze(-1)
    h, ent = st["d_entropy"].unsqueeze(-1), out["entropy"].unsqueeze(-1)
    grad = torch.where(p > 0, -p * (g + h * (lp + ent)), torch.zeros_like(p))
    grad.scatter_add_(-1, st["targets"].clamp(min=0).unsqueeze(-1), g)
    out["grad"] = (grad / temp).to(x.dtype)
    return out


def _plain_teacher(st):
    t = st["values"] / st["case"]["temperature"]
    d, log_s = _plain_softmax(t)
    log_q = d - log_s
    return log_q.exp(), log_q


# ------------------------------------------------------------------ the framework's calls
def _run_own(st):
    from mamba_tp_lite_b200 import logprobs as P

    case = st["case"]
    temp = case["temperature"]
    if case["op"] == "score":
        r = P.lm_head_logprobs(st["hidden"], st["weight"], st["targets"], temperature=temp)
        return {"logprob": r.logprob, "entropy": r.entropy}
    if case["op"] == "logprobs":
        r = P.token_logprobs(st["logits"], st["targets"], top_k=case["top_k"], temperature=temp)
        out = {"logprob": r.logprob, "entropy": r.entropy}
        if case["top_k"]:
            out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
        return out
    if case["op"] == "distill":
        if case["grad"] == "none":
            return {"loss": P.distill_topk_loss(st["logits"], st["ids"], st["values"], temperature=temp)}
        if case["grad"] == "joint":
            loss, grad = P.distill_topk_loss_and_grad(st["logits"], st["ids"], st["values"], st["weight"],
                                                      temperature=temp)
            return {"loss": loss, "grad": grad}
        x = st["logits"].detach().requires_grad_()
        loss = P.distill_topk_loss(x, st["ids"], st["values"], temperature=temp)
        (grad,) = torch.autograd.grad([loss], [x], [st["weight"]])
        return {"loss": loss.detach(), "grad": grad}
    x = st["logits"].detach().requires_grad_()
    r = P.token_logprobs(x, st["targets"], temperature=temp)
    (grad,) = torch.autograd.grad([r.logprob, r.entropy], [x], [st["d_logprob"], st["d_entropy"]])
    return {"logprob": r.logprob.detach(), "entropy": r.entropy.detach(), "grad": grad}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    v, temp = case["vocab"], case["temperature"]
    if case["op"] == "score":
        src = st["hidden"]
        weight = st["weight"].double()
    else:
        src = st["logits"]
    lead = src.shape[:-1]
    index = [(i, j) for i in range(lead[0]) for j in range(0, lead[1], 1024)]
    parts = []
    for i, j in index:
        sl = (i, slice(j, min(j + 1024, lead[1])))
        x = src[sl].double()
        z = (x @ weight.T if case["op"] == "score" else x) / temp
        lse = torch.logsumexp(z, -1)
        part = {}
        if case["op"] == "distill":
            t = st["values"][sl].double() / temp
            q = torch.softmax(t, -1)
            pz = torch.exp(z - lse[:, None])
            lp = torch.take_along_dim(z, st["ids"][sl], -1) - lse[:, None]
            part["loss"] = (q * (t - torch.logsumexp(t, -1, keepdim=True) - lp)).sum(-1)
            if case["grad"] != "none":
                target = torch.zeros_like(z).scatter_add_(-1, st["ids"][sl], q)
                part["grad"] = (pz - target) * (st["weight"][sl].double()[:, None] / temp)
            parts.append(part)
            continue
        tgt = st["targets"][sl]
        rows = torch.arange(tgt.shape[0], device=tgt.device)
        used = tgt >= 0
        part["logprob"] = torch.where(used, z[rows, tgt.clamp(min=0)] - lse, 0.0)
        p = torch.exp(z - lse[:, None])
        logp = (z - lse[:, None]).clamp(min=-1e300)  # a banned token has p = 0 and adds nothing
        part["entropy"] = -(p * logp).sum(-1)
        if case.get("top_k") and case["op"] == "logprobs":
            top = torch.sort(x, dim=-1, descending=True, stable=True)
            part["top_ids"] = top.indices[:, :case["top_k"]]
            part["top_logprobs"] = top.values[:, :case["top_k"]] / temp - lse[:, None]
        if case["op"] == "logprobs_grad":
            g = torch.where(used, st["d_logprob"][sl].double(), 0.0)
            h = st["d_entropy"][sl].double()
            onehot = torch.zeros_like(z)
            onehot[rows, tgt.clamp(min=0)] = 1.0
            part["grad"] = (g[:, None] * (onehot - p) - h[:, None] * p * (logp + part["entropy"][:, None])) / temp
        parts.append(part)
    return {name: torch.cat([part[name] for part in parts]).view(*lead, *parts[0][name].shape[1:])
            for name in parts[0]}


def work(case):
    rows, v = _rows(case), case["vocab"]
    if case["op"] == "score":
        h = case["hidden"]
        return {"bytes": 2 * (rows * h + v * h) + rows * 16, "flops": 2 * rows * v * h}
    es = _SIZE[case["dtype"]]
    read = rows * v * es
    if case["op"] == "logprobs":
        return {"bytes": read + rows * (16 + 12 * case["top_k"]), "flops": 6 * rows * v}
    if case["op"] == "logprobs_grad":
        return {"bytes": 2 * read + rows * 24, "flops": 12 * rows * v}
    k = case["top_k"]
    if case["grad"] == "none":
        return {"bytes": read + rows * (4 + 12 * k), "flops": 4 * rows * v}
    return {"bytes": 2 * read + rows * (8 + 12 * k), "flops": 8 * rows * v}
