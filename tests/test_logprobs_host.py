"""The operators on logits without a GPU: refusals, row layouts, and the 64-bit reference the GPU tests use
against torch and against differences.  No kernel is launched here."""
import ctypes as C

import numpy as np
import pytest
import torch

from mamba_tp_lite_b200 import _lib as L
from mamba_tp_lite_b200 import logprobs as P
from mamba_tp_lite_b200 import quant_eval
from tests import logits_ref as R


# ------------------------------------------------------------------ the 64-bit reference
def _rows(rows, v, seed, scale=3.0):
    return np.random.default_rng(seed).standard_normal((rows, v)) * scale


def test_reference_log_probabilities_match_torch():
    x = _rows(7, 33, 0)
    t = np.array([0, 5, 32, -1, 7, 33, 2])
    lp = torch.log_softmax(torch.from_numpy(x) / 0.7, -1)
    np.testing.assert_allclose(R.log_probs(x, 0.7), lp.numpy(), atol=1e-12)
    got = R.token_logprob(x, t, 0.7)
    assert got[3] == 0 and np.isnan(got[5])
    np.testing.assert_allclose(got[[0, 1, 2, 4, 6]], lp.numpy()[[0, 1, 2, 4, 6], t[[0, 1, 2, 4, 6]]], atol=1e-12)
    np.testing.assert_allclose(R.entropy(x, 0.7), -(lp.exp() * lp).sum(-1).numpy(), atol=1e-12)


def test_reference_top_orders_ties_nan_and_zeros():
    x = np.array([[1.0, 2.0, 2.0, np.nan, -np.inf, np.inf, 0.0, -0.0]])
    assert R.top(x, 8).tolist() == [[3, 5, 1, 2, 0, 6, 7, 4]]


def test_reference_empty_row():
    x = np.full((1, 5), -np.inf)
    assert R.token_logprob(x, np.array([2]))[0] == -np.inf and R.entropy(x)[0] == 0
    grad, _ = R.token_logprobs_grad(x, np.array([2]), [1.0], [1.0])
    assert (grad == 0).all()


@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_reference_gradients_match_differences(temperature):
    x = _rows(3, 9, 1)
    t = np.array([4, -1, 8])
    g, h = np.array([0.7, 0.3, -1.1]), np.array([0.2, -0.4, 0.0])
    ids = np.array([[1, 4, 4, -1], [0, 3, 8, 2], [-1, -1, -1, -1]])
    vals = _rows(3, 4, 2)
    w = np.array([0.5, 1.5, 2.0])
    grad, _ = R.token_logprobs_grad(x, t, g, h, temperature)
    dgrad, _ = R.distill_grad(x, ids, vals, w, temperature)
    eps = 1e-6
    for r in range(3):
        for j in range(9):
            hi, lo = x.copy(), x.copy()
            hi[r, j] += eps
            lo[r, j] -= eps
            f = lambda y: (g * R.token_logprob(y, t, temperature) + h * R.entropy(y, temperature)).sum()
            assert abs((f(hi) - f(lo)) / (2 * eps) - grad[r, j]) < 1e-8
            f = lambda y: (w * R.distill_loss(y, ids, vals, temperature)).sum()
            assert abs((f(hi) - f(lo)) / (2 * eps) - dgrad[r, j]) < 1e-8


def test_reference_distillation_is_zero_at_the_teacher():
    x = _rows(4, 12, 3)
    ids = np.argsort(-x, -1)
    loss = R.distill_loss(x, ids, np.take_along_axis(x, ids, 1))
    np.testing.assert_allclose(loss, 0, atol=1e-12)


# ------------------------------------------------------------------ row layouts
LAYOUTS = {
    "rows": lambda: torch.randn(6, 11),
    "one": lambda: torch.randn(11),
    "batch": lambda: torch.randn(2, 3, 11),
    "shifted": lambda: torch.randn(2, 4, 11)[:, :-1],
    "cut": lambda: torch.randn(2, 4, 16)[..., :11],
    "cut_and_shifted": lambda: torch.randn(3, 5, 16)[:, 1:, 2:13],
    "deep": lambda: torch.randn(2, 3, 4, 11)[:, :, :-1],
    "three_strides": lambda: torch.randn(4, 6, 8, 11)[:3, :5, :7],
    "columns": lambda: torch.randn(11, 6).t(),
    "expanded": lambda: torch.randn(1, 11).expand(5, 11),
    "expanded_batch": lambda: torch.randn(1, 3, 11).expand(4, 3, 11),
    "transposed": lambda: torch.randn(3, 4, 11).transpose(0, 1),
    "empty": lambda: torch.randn(0, 3, 11),
    "every_other": lambda: torch.randn(8, 11)[::2],
}


@pytest.mark.parametrize("name", LAYOUTS)
def test_row_layout_addresses_every_row(name):
    x = LAYOUTS[name]()
    y, outer, inner, ld_outer, ld = P._row_layout(x)
    v = x.shape[-1]
    assert outer * inner == x.numel() // v
    want = x.reshape(-1, v)
    base = y.storage_offset()
    flat = torch.as_strided(y, (y.untyped_storage().nbytes() // 4,), (1,), 0)
    for o in range(outer):
        for i in range(inner):
            at = base + o * ld_outer + i * ld
            assert torch.equal(flat[at:at + v], want[o * inner + i])


@pytest.mark.parametrize("name", [n for n in LAYOUTS if n != "empty"])
def test_gradient_layout_is_apart_and_addressed(name):
    x = LAYOUTS[name]()
    x, outer, inner, ld_outer, ld = P._row_layout(x)
    grad, g_outer, g_ld = P._grad_like(x, inner, ld_outer, ld)
    v = x.shape[-1]
    assert grad.shape == x.shape and grad.dtype == x.dtype
    base = grad.storage_offset()
    flat = torch.as_strided(grad, (grad.untyped_storage().nbytes() // 4,), (1,), 0)
    seen = set()
    for o in range(outer):
        for i in range(inner):
            at = base + o * g_outer + i * g_ld
            span = set(range(at, at + v))
            assert not span & seen and max(span) < flat.numel()
            seen |= span
            flat[at:at + v] = float(o * inner + i)
    assert torch.equal(grad.reshape(-1, v), torch.arange(float(outer * inner))[:, None].expand(-1, v))


# ------------------------------------------------------------------ refusals
def test_no_cpu_path():
    x = torch.randn(2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.token_logprobs(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        P.distill_topk_loss(x, torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        P.lm_head_logprobs(x, torch.randn(5, 8), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        quant_eval.record_top_logits(torch.randn(1, 2, 80))


def test_argument_checks():
    x = torch.randn(2, 3, 8)
    ids = torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(TypeError, match="integers"):
        P._check_ids(ids.float(), x.shape[:-1], x.device, "f", "targets")
    with pytest.raises(TypeError, match="integers"):
        P._check_ids(ids.bool(), (2, 3), x.device, "f", "targets")
    with pytest.raises(ValueError, match="shape"):
        P._check_ids(ids, (2, 4), x.device, "f", "targets")
    with pytest.raises(ValueError, match="are on cpu"):
        P._check_ids(ids, (2, 3), torch.device("cuda:0"), "f", "targets")
    for k in (-1, 9, 129):
        with pytest.raises(ValueError, match="top_k"):
            P._check_top_k(k, 8 if k < 100 else 1000, "f")
    for t in (0.0, -1.0, 1e-40, 1e30, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            P._check_temperature(t, "f")
    with pytest.raises(ValueError, match="shape"):
        P._check_rows(torch.zeros(2), (2, 3), x.device, "f", "row_weight")
    with pytest.raises(TypeError, match="floating"):
        P._check_rows(ids, (2, 3), x.device, "f", "row_weight")
    for shape in ((2, 3), (2, 3, 0), (2, 3, 129), (2, 4, 5)):
        with pytest.raises(ValueError, match="teacher ids"):
            P._teacher(x, torch.zeros(shape, dtype=torch.int64), torch.zeros(shape), "f")
    with pytest.raises(ValueError, match="teacher logits"):
        P._teacher(x, torch.zeros(2, 3, 5, dtype=torch.int64), torch.zeros(2, 3, 4), "f")


def _refused(name, *args, code=L.MTP_ERR_ARG, text=""):
    lib = L.load()
    assert getattr(lib, name)(*args) == code
    assert text in lib.mtp_last_error().decode()


def test_c_entry_points_refuse_bad_arguments():
    """Host checks, before any CUDA call: the pointers are never used."""
    p = 4096
    tok = lambda dt=L.F32, outer=1, inner=4, ldo=0, ld=64, v=64, t=1.0, tgt=p, k=0, ids=None, tl=None, x=p: (
        "mtp_token_logprobs", x, dt, outer, inner, ldo, ld, v, tgt, t, p, p, None, k, ids, tl, None)
    _refused(*tok(x=None), text="null pointer")
    _refused(*tok(dt=7), code=L.MTP_ERR_UNSUPPORTED, text="dtype")
    _refused(*tok(v=0), text="vocabulary")
    _refused(*tok(v=(1 << 30) + 1), text="vocabulary")
    _refused(*tok(outer=-1), text="sizes")
    _refused(*tok(ld=-64), text="sizes")
    _refused(*tok(outer=1 << 20, inner=1 << 20), text="rows")
    _refused(*tok(t=0.0), text="temperature")
    _refused(*tok(t=float("nan")), text="temperature")
    _refused(*tok(tgt=None), text="targets")
    _refused(*tok(k=129, ids=p, tl=p), text="top_k")
    _refused(*tok(k=65, ids=p, tl=p), text="top_k")
    _refused(*tok(k=5), text="top_ids")
    assert L.load().mtp_token_logprobs(None, L.F32, 0, 4, 0, 64, 64, None, 1.0, None, None, None, 0, None, None,
                                       None) == L.MTP_OK  # no rows: nothing to do
    bwd = lambda ent=p, dlp=p, dent=p, gld=64, tgt=p, stats=p: (
        "mtp_token_logprobs_bwd", p, L.F32, 1, 4, 0, 64, 64, tgt, 1.0, stats, ent, dlp, dent, p, 0, gld, None)
    _refused(*bwd(ent=None), text="entropy")
    _refused(*bwd(tgt=None), text="targets")
    _refused(*bwd(gld=63))
    _refused(*bwd(stats=None))
    dis = lambda k=4, vdt=L.F32, ids=p, loss=p: (
        "mtp_distill_topk", p, L.F32, 1, 4, 0, 64, 64, ids, p, vdt, k, 1.0, loss, None, None)
    _refused(*dis(k=0), text="k must")
    _refused(*dis(k=129), text="k must")
    _refused(*dis(vdt=9), text="values")
    _refused(*dis(ids=None))
    _refused(*dis(loss=None))
    dg = lambda k=4, w=p, gld=64: ("mtp_distill_topk_grad", p, L.F32, 1, 4, 0, 64, 64, p, p, L.F32, k, 1.0, None, w,
                                   None, p, 0, gld, None)
    _refused(*dg(k=129), text="k must")
    _refused(*dg(w=None))
    _refused(*dg(gld=1))
    n = C.c_int64(0)
    _refused("mtp_lm_head_logprobs_workspace", p, 32, 4, 32, p, 32, 64, L.F16, 0, C.byref(n), text="dtype")
    _refused("mtp_lm_head_logprobs_workspace", p, 32, -1, 32, p, 32, 64, L.BF16, 0, C.byref(n))
    assert L.load().mtp_lm_head_logprobs_workspace(p, 32, 4, 32, p, 32, 64, L.BF16, 0, C.byref(n)) == L.MTP_OK and n.value > 0
    lm = lambda ws=p, nb=n.value, ldh=32, dt=L.BF16, tgt=p, k=0: (
        "mtp_lm_head_logprobs", p, ldh, 4, 32, p, 32, 64, dt, tgt, 1.0, p, p, k, None, None, ws, nb, None)
    _refused(*lm(ws=None), text="null")
    _refused(*lm(nb=n.value - 1), text="workspace")
    _refused(*lm(ws=4104), text="workspace")
    _refused(*lm(ldh=31))
    _refused(*lm(dt=L.F16), text="dtype")
    _refused(*lm(tgt=None), text="targets")
    _refused(*lm(k=3), text="top_ids")


# ------------------------------------------------------------------ calls, on a library that only records them
class Recorder:
    """In place of the library: the calls' names and arguments, and whether the device was set around each."""

    def __init__(self, monkeypatch):
        self.calls, self.depth = [], 0
        monkeypatch.setattr(L, "require_cuda", lambda t, what: None)
        monkeypatch.setattr(L, "stream_ptr", lambda stream=None: 0)
        monkeypatch.setattr(L, "call", self.call)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)  # a CPU tensor's device has no index: another one
        monkeypatch.setattr(torch.cuda, "device", self.device)

    def call(self, name, *args):
        self.calls.append((name, args, self.depth))

    def device(self, dev):
        rec = self

        class Guard:
            def __enter__(self):
                rec.depth += 1

            def __exit__(self, *exc):
                rec.depth -= 1

        return Guard()


def test_every_call_is_made_on_the_device_of_its_tensors(monkeypatch):
    """The workspace depends on the number of SMs, so its size is asked for on that device too."""
    rec = Recorder(monkeypatch)
    x, t = torch.randn(4, 16), torch.zeros(4, dtype=torch.int64)
    P.token_logprobs(x, t)
    P.distill_topk_loss(x, t[:, None], torch.zeros(4, 1))
    P.lm_head_logprobs(x, torch.randn(9, 16), t, top_k=2)
    assert [c[0] for c in rec.calls] == ["mtp_token_logprobs", "mtp_distill_topk", "mtp_lm_head_logprobs_workspace",
                                         "mtp_lm_head_logprobs"]
    assert all(depth == 1 for _, _, depth in rec.calls)


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """A dual tensor that does not require a gradient must not come back without its tangent."""
    rec = Recorder(monkeypatch)
    t = torch.zeros(4, dtype=torch.int64)
    w = torch.randn(9, 16)
    with torch.autograd.forward_ad.dual_level():
        x = torch.autograd.forward_ad.make_dual(torch.randn(4, 16), torch.ones(4, 16))
        dw = torch.autograd.forward_ad.make_dual(w, torch.ones(9, 16))
        for call in (lambda: P.token_logprobs(x, t), lambda: P.distill_topk_loss(x, t[:, None], torch.zeros(4, 1)),
                     lambda: P.distill_topk_loss_and_grad(x, t[:, None], torch.zeros(4, 1), torch.ones(4)),
                     lambda: P.lm_head_logprobs(x, w, t), lambda: P.lm_head_logprobs(torch.randn(4, 16), dw, t)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert not rec.calls
        P.token_logprobs(torch.randn(4, 16), t)  # no dual tensor: as ever
    assert len(rec.calls) == 1


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("entropy", [False, True])
def test_the_entropy_is_computed_only_where_it_is_asked_for(monkeypatch, requires_grad, entropy):
    rec = Recorder(monkeypatch)
    x = torch.randn(4, 16, requires_grad=requires_grad)
    r = P.token_logprobs(x, torch.zeros(4, dtype=torch.int64), entropy=entropy)
    assert (r.entropy is not None) == entropy
    if requires_grad:
        r.logprob.sum().backward()
    for name, args, _ in rec.calls:
        assert (args[10] is not None) == entropy  # where the forward call writes it, and the backward call reads it


def test_sequence_nll_of_padded_sequences(monkeypatch):
    """Partly padded, padded after the first token, and sequences of one token: nothing to predict counts 0."""
    monkeypatch.setattr(quant_eval, "token_logprobs", lambda x, t, entropy: P.TokenLogprobs(
        torch.from_numpy(R.token_logprob(x.double().numpy().reshape(-1, x.shape[-1]), t.numpy().reshape(-1))).view(t.shape),
        None, None, None))
    g = torch.Generator().manual_seed(0)
    logits = torch.randn(3, 5, 11, generator=g, dtype=torch.float64)
    ids = torch.tensor([[1, 2, 3, 4, 5], [6, 7, -1, -1, -1], [8, -1, -1, -1, -1]])
    lp = torch.log_softmax(logits, -1)
    want = [-(lp[0, 0, 2] + lp[0, 1, 3] + lp[0, 2, 4] + lp[0, 3, 5]) / 4, -lp[1, 0, 7], torch.tensor(0.0)]
    got = quant_eval.sequence_nll(logits, ids)
    np.testing.assert_allclose(got.numpy(), torch.stack([w.double() for w in want]).numpy(), atol=1e-12)
    assert (quant_eval.sequence_nll(logits[:, :1], ids[:, :1]) == 0).all()


# ------------------------------------------------------------------ whether a test of scoring can fail
def _truncated_sum(h, w, step=16):
    """h . w^T in 24 bits, cut off after every `step` products."""
    acc = np.zeros((h.shape[0], w.shape[0]))
    for k in range(0, h.shape[1], step):
        acc = acc + h[:, k:k + step] @ w[:, k:k + step].T
        ulp = 2.0 ** (np.floor(np.log2(np.abs(acc))) - 23)
        acc = np.trunc(acc / ulp) * ulp
    return acc


@pytest.mark.parametrize("rows,v,k", [(6, 777, 1024), (5, 2049, 2048), (4, 1001, 1100), (4, 1001, 2560), (3, 4001, 3000)])
def test_exact_hidden_states_show_a_loss_of_precision(rows, v, k):
    """The mistakes that scoring must not make, made here: each goes past the bounds that the GPU is held to."""
    h, w = R.exact_score_inputs(rows, v, k, k)
    for a in (h, w):
        assert torch.equal(torch.from_numpy(a).bfloat16().double(), torch.from_numpy(a))
    n = R.score_accumulators(k)
    assert n <= 1024
    for k0 in range(0, k, n):  # exact in every accumulator: so says the same sum cut off at every step
        part = h[:, k0:k0 + n] @ w[:, k0:k0 + n].T
        assert (part < R.SUM_LIMIT).all() and (part % R.SUM_GRAIN == 0).all()
        assert (_truncated_sum(h[:, k0:k0 + n], w[:, k0:k0 + n]) == part).all()
    t = np.arange(rows) % v
    x, lp, lp_bound, ent, ent_bound = R.exact_score_bounds(h, w, t, n if k > n else None)

    def seen(y):
        return (np.abs(R.token_logprob(y, t) - lp) > lp_bound).all()

    assert not seen(x)
    assert seen(torch.from_numpy(x).bfloat16().double().numpy())  # logits in bf16
    gone = x.copy()
    gone[:, 512:528] = -np.inf
    assert seen(gone)                                              # sixteen tokens passed over
    if k > n:
        assert seen(_truncated_sum(h, w))                          # one accumulator for all of K
        assert seen(x - h[:, n:n + 16] @ w[:, n:n + 16].T)         # sixteen positions of K passed over
