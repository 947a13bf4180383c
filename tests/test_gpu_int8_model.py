"""A model with int8 linears: each 8-bit call of a forward pass against its definition in 64 bits on the inputs that it got,
and what lies between them against a plain forward in 64 bits."""
import pytest
import torch
import torch.nn.functional as F

from mamba_tp_lite_b200 import _mixer, model as model_file
from mamba_tp_lite_b200 import int8 as Q
from mamba_tp_lite_b200.config import MambaConfig
from mamba_tp_lite_b200.cuda_graph import GraphedStepper
from mamba_tp_lite_b200.model import LayerCache, MambaCache, MambaLM
from tests import int8_ref as R
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def build(dtype, bias=False, d_model=48, n_layer=3, seed=0, d_state=16):
    cfg = MambaConfig(d_model=d_model, n_layer=n_layer, vocab_size=200, d_state=d_state, dt_rank=8, bias=bias)
    g = torch.Generator().manual_seed(seed)
    m = MambaLM(cfg)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if name.endswith("norm.weight") or name.endswith("norm_f.weight"):
                p.copy_(1 + 0.2 * torch.randn(p.shape, generator=g))
            elif name.endswith("dt_proj.bias"):
                p.copy_(torch.rand(p.shape, generator=g) - 3)
            elif "A_log" not in name and not name.endswith(".D"):
                p.copy_(torch.randn(p.shape, generator=g) * (1.0 if p.dim() < 2 else p.shape[-1] ** -0.5))
    return m.to(dev()).to(dtype).eval()


class Calls:
    """The 8-bit calls of a forward pass with copies of what they got and gave, in order."""

    def __init__(self, monkeypatch):
        self.made = []
        for module, names in ((_mixer, ("int8_linear", "quantize_rows")), (model_file, ("rms_norm_int8", "add_rms_norm_int8"))):
            for name in names:
                monkeypatch.setattr(module, name, self.wrap(name, getattr(Q, name)))

    def wrap(self, name, fn):
        def call(*args, **kw):
            def copy(v):
                if isinstance(v, torch.Tensor):
                    return v.clone()
                return type(v)(*map(copy, v)) if isinstance(v, Q.Int8Rows) else tuple(map(copy, v)) if isinstance(v, tuple) else v

            before = tuple(copy(a) for a in args)
            out = fn(*args, **kw)
            self.made.append((name, before, kw, copy(out)))
            return out

        return call

    def take(self, name):
        got = self.made.pop(0)
        assert got[0] == name
        return got[1:]


def mix(m, xz, conv, ssm):
    """conv1d, x_proj, dt_proj, the scan and the gate in 64 bits: (y [b, l, e], conv state, ssm state)."""
    d = lambda t: t.detach().double()
    e, n, r, k = m.es, m.cfg.d_state, m.cfg.dt_rank, m.cfg.d_conv
    x, z = d(xz).split(e, -1)
    wide = torch.cat([d(conv).transpose(1, 2), x], 1)
    c = F.silu(sum(wide[:, i:i + x.shape[1]] * d(m.conv1d.weight)[:, 0, i] for i in range(k)) + d(m.conv1d.bias))
    low, B, C = (c @ d(m.x_proj.weight).T).split([r, n, n], -1)
    dt = F.softplus(low @ d(m.dt_proj.weight).T + d(m.dt_proj.bias))
    A, h, ys = -torch.exp(d(m.A_log)), d(ssm), []
    for t in range(x.shape[1]):
        h = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * c[:, t])[..., None] * B[:, t, None, :]
        ys.append((h * C[:, t, None, :]).sum(-1) + d(m.D) * c[:, t])
    return torch.stack(ys, 1) * F.silu(z), wide[:, -(k - 1):].transpose(1, 2), h


def through(stages):
    """What a generator returns."""
    while True:
        try:
            next(stages)
        except StopIteration as done:
            return done.value


def same_rows(a, b):
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scale, b.scale)


def follow(model, calls, ids, logits, before, after, step=False):
    """Goes through the recorded calls of one pass over ids [b, l]."""
    b, l = ids.shape
    cfg, wtype = model.cfg, model.embedding.weight.dtype
    tol = dict(rtol=2e-4, atol=2e-5)
    resid = model.embedding.weight.detach()[ids.reshape(-1)].float()
    (x, w, eps), _, rows = calls.take("rms_norm_int8")
    assert torch.equal(x, resid) and torch.equal(w, model.layers[0].norm.weight) and eps == cfg.layer_norm_epsilon
    R.check_rows(rows.codes, rows.scale, R.norm(resid, w, eps))
    for i, layer in enumerate(model.layers):
        m = layer.mixer
        (x, wq, bias), kw, xz = calls.take("int8_linear")
        same_rows(x, rows)
        same_rows(wq, Q.quantize_rows(m.in_proj.weight.detach()))
        assert (bias is None) == (m.in_proj.bias is None) and kw == dict(dtype=wtype)
        assert torch.equal(xz, R.linear(x.codes, x.scale, wq.codes, wq.scale, m.in_proj.bias, wtype))
        # each code is off by half a step at most: what that makes of the product with the model's own weight
        x64, w64 = R.norm(resid, layer.norm.weight, cfg.layer_norm_epsilon), m.in_proj.weight.detach().double()
        sx, sw = x.scale.double()[:, None] / 2, wq.scale.double()[:, None] / 2
        bound = sx @ w64.abs().sum(1)[None] + x64.abs().sum(1)[:, None] @ sw.T + w64.shape[1] * sx @ sw.T
        exact = x64 @ w64.T + (0 if bias is None else bias.double())
        rounding = exact.abs() * (torch.finfo(wtype).eps / 2 + 4 * R.U) + bound * 2.0 ** -7
        assert ((xz.double() - exact).abs() <= bound + rounding).all()
        (got,), _, rows = calls.take("quantize_rows")
        old, new = before.layers[i], after.layers[i]
        if wtype == torch.float32:
            y, conv, ssm = mix(m, xz.view(b, l, -1), old.conv_state, old.ssm_state)
            torch.testing.assert_close(got.double().view(b, l, -1), y, **tol)
            torch.testing.assert_close(new.conv_state.double(), conv, rtol=0, atol=0)
            torch.testing.assert_close(new.ssm_state.double(), ssm, **tol)
        else:  # what a model without int8 linears makes of this xz, to the bit
            conv, ssm = old.conv_state.clone(), old.ssm_state.clone()
            if step:
                y = m._step_mix(xz, conv, ssm)
            else:
                y, conv, ssm = through(m._prefill_mix(xz, b, l, conv, ssm))
            assert torch.equal(got, y) and torch.equal(new.conv_state, conv) and torch.equal(new.ssm_state, ssm)
        R.check_rows(rows.codes, rows.scale, got)
        (x, wq, bias), kw, branch = calls.take("int8_linear")
        same_rows(x, rows)
        same_rows(wq, Q.quantize_rows(m.out_proj.weight.detach()))
        assert kw == dict(dtype=torch.float32)
        assert torch.equal(branch, R.linear(x.codes, x.scale, wq.codes, wq.scale, m.out_proj.bias, torch.float32))
        if i + 1 < cfg.n_layer:
            (x, r, w, eps), kw, (rows, h) = calls.take("add_rms_norm_int8")
            assert torch.equal(x, branch) and torch.equal(r, resid) and torch.equal(w, model.layers[i + 1].norm.weight)
            assert kw == dict(inplace=True) and torch.equal(h, R.add(branch, resid))
            R.check_rows(rows.codes, rows.scale, R.norm(h, w, eps))
            resid = h
    assert not calls.made
    last = R.norm(R.add(branch, resid), model.norm_f.weight, cfg.layer_norm_epsilon)
    # the norm rounded to the model's type, a sum of d products and the result rounded again, u being half a step of that
    # type; the norm's and the product's fp32 sums are off by less than 2 d + 16 half steps of fp32
    emb, u = model.embedding.weight.detach().double(), torch.finfo(wtype).eps / 2
    want, size = last @ emb.T, last.abs() @ emb.abs().T
    bound = (u + (2 * cfg.d_model + 16) * R.U) * size * (1 + u) + u * want.abs()
    assert ((logits.view(b * l, -1).double() - want).abs() <= bound).all()


def copy_of(cache):
    return MambaCache([LayerCache(c.conv_state.clone(), c.ssm_state.clone()) for c in cache.layers])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("b,l", [(1, 1), (2, 9), (3, 70)])
def test_prefill_and_steps(monkeypatch, dtype, bias, b, l):
    model = build(dtype, bias)
    model.quantize_linears()
    calls = Calls(monkeypatch)
    ids = torch.randint(0, 200, (b, l + 3), generator=torch.Generator().manual_seed(1)).to(dev())
    zero = MambaCache.allocate(model.cfg, b, dev(), dtype)
    logits, cache = model.prefill(ids[:, :l])
    follow(model, calls, ids[:, :l], logits, zero, cache)
    for t in range(l, l + 2):
        before = copy_of(cache)
        logits = model.step(ids[:, t:t + 1], cache)
        follow(model, calls, ids[:, t:t + 1], logits, before, cache, step=True)
    before = copy_of(cache)
    logits, more = model.prefill(ids[:, 1:], cache)  # a prompt goes on from a cache
    follow(model, calls, ids[:, 1:], logits, before, more)


def test_off_again_and_what_stays(monkeypatch):
    model = build(torch.bfloat16, d_model=64)
    ids = torch.randint(0, 200, (2, 20), generator=torch.Generator().manual_seed(1)).to(dev())
    names = list(model.state_dict())
    plain, cache = model.prefill(ids)
    step = model.step(ids[:, :1], copy_of(cache))
    model.quantize_linears()
    q, _ = model.prefill(ids)
    assert not torch.equal(q, plain) and list(model.state_dict()) == names
    model.quantize_linears(False)
    calls = Calls(monkeypatch)
    again, cache2 = model.prefill(ids)
    assert torch.equal(again, plain) and not calls.made
    assert torch.equal(model.step(ids[:, :1], cache2), step)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b", [1, 3, 20])
def test_generate_graphs_and_scores(dtype, b):
    model = build(dtype, d_model=64)
    model.quantize_linears()
    ids = torch.randint(0, 200, (b, 12), generator=torch.Generator().manual_seed(b)).to(dev())
    eager = model.generate(ids, 6)
    assert torch.equal(model.generate(ids, 6, graphed=True), eager)
    logits, cache = model.prefill(ids)
    stepper = GraphedStepper(model, cache, b, "cuda")
    twin = copy_of(cache)
    stepper.capture()
    for t in range(4):
        got = stepper.replay(ids[:, t:t + 1])
        assert torch.equal(got, model.step(ids[:, t:t + 1], twin))
    for c, d in zip(cache.layers, twin.layers):
        assert torch.equal(c.ssm_state, d.ssm_state) and torch.equal(c.conv_state, d.conv_state)
    stepper.release()
    r, _ = model.score(ids)
    want = torch.log_softmax(logits.double(), -1)[:, :-1].gather(2, ids[:, 1:, None])[..., 0]
    # the prefill's logits are rounded to the model's type: half a step of the largest, twice (the token's and the sum's)
    off = 2 * logits.double().abs().max() * torch.finfo(dtype).eps / 2 + 2e-5
    assert ((r.logprob[:, :-1].double() - want).abs() <= off).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_mixer_by_itself(dtype):
    model = build(dtype, bias=True)
    model.quantize_linears()
    m = model.layers[1].mixer
    x = torch.randn(2, 7, 48, generator=torch.Generator().manual_seed(3)).to(dev()).to(dtype)
    out, conv, ssm = m.prefill(x)
    rows = Q.quantize_rows(x.view(-1, 48))
    branch, conv2, ssm2 = m._prefill_int8(rows, 2, 7, None, None)
    assert out.dtype == dtype and torch.equal(out, branch.to(dtype).view(2, 7, 48))
    assert torch.equal(conv, conv2) and torch.equal(ssm, ssm2)
    cache = LayerCache(conv, ssm)
    y = m.step(x[:, 0], cache)
    assert y.shape == (2, 48) and y.dtype == dtype and torch.isfinite(y.float()).all()
