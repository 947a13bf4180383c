"""The 8-bit linear path without a GPU: which calls in place are taken, and that a model's int8 weights are those of its
parameters."""
import copy
import io

import pytest
import torch

from mamba_tp_lite_b200 import _mixer, model as model_file
from mamba_tp_lite_b200 import int8 as Q
from mamba_tp_lite_b200.config import MambaConfig
from mamba_tp_lite_b200.model import MambaCache, MambaLM
from tests.test_logprobs_host import Recorder


def test_in_place_beside_x_in_three_dimensions(monkeypatch):
    rec = Recorder(monkeypatch)
    buf, w = torch.randn(2, 3, 48), torch.ones(16)
    for x, res in [(buf[:, :, :16], buf[:, :, 16:32]), (buf[:, :, 32:], buf[:, :, :16]), (buf[0], buf[1])]:
        weight = torch.ones(x.shape[-1])
        assert Q.add_rms_norm_int8(x, res, weight, inplace=True)[1] is res
        name, args, _ = rec.calls.pop()
        assert args[0] == x.data_ptr() and args[3] == args[6] == res.data_ptr() and args[2] == args[5] == args[7] == 48
    # x is copied before the residual is written
    x = buf.transpose(0, 1)[:, :, :16]
    Q.add_rms_norm_int8(x, buf.view(6, 48).view(3, 2, 48)[:, :, :16], w, inplace=True)
    assert rec.calls.pop()[1][0] != x.data_ptr()
    rows = buf.view(6, 48)
    for x, res in [(buf[:, :, :16], buf[:, :, 15:31]), (buf[:, :, :16], buf[:, :, :16]), (rows[:5, 32:], rows[1:, :16].as_strided((5, 16), (48, 1), 47)),
                   (buf[:, :, :16], buf.view(-1)[16:112].view(2, 3, 16))]:
        with pytest.raises(ValueError, match="share memory"):
            Q.add_rms_norm_int8(x, res, w, inplace=True)
    assert not rec.calls


# ------------------------------------------------------------------ weights that change after they were quantised
class Through(Exception):
    """Raised in place of the first call of a pass: the weights were taken."""


def small_model(monkeypatch, n_layer=2):
    rec = Recorder(monkeypatch)
    lm = MambaLM(MambaConfig(d_model=64, n_layer=n_layer, vocab_size=64, dt_rank=8)).bfloat16()
    lm.quantize_linears()
    return lm, rec


def passes(lm):
    """Every way into the int8 linears."""
    ids, x = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    cache = MambaCache.allocate(lm.cfg, 2, "cpu", torch.bfloat16)
    m = lm.layers[-1].mixer
    return [lambda: lm.prefill(ids), lambda: lm.prefill(ids, cache), lambda: lm.step(ids[:, :1], cache), lambda: lm.score(ids),
            lambda: m.prefill(x), lambda: m(x), lambda: m.step(x[:, 0], cache.layers[-1])]


def taken(lm, rec, monkeypatch):
    """Whether the passes take the model's int8 weights; each is stopped at its first 8-bit call."""
    def stop(*args, **kw):
        raise Through

    monkeypatch.setattr(_mixer, "quantize_rows", stop)
    monkeypatch.setattr(model_file, "rms_norm_int8", stop)
    got = []
    for run in passes(lm):
        try:
            run()
        except Through:
            got.append(True)
        except RuntimeError as e:
            assert "quantize_linears" in str(e) and "layer " in str(e)
            got.append(False)
    monkeypatch.setattr(_mixer, "quantize_rows", Q.quantize_rows)
    monkeypatch.setattr(model_file, "rms_norm_int8", Q.rms_norm_int8)
    assert all(got) or not any(got)
    return got[0]


def double(lm):
    return {k: 2 * v for k, v in lm.state_dict().items()}


def a_new_parameter(lm):
    lm.layers[1].mixer.out_proj.weight = torch.nn.Parameter(lm.layers[1].mixer.out_proj.weight.detach().clone())


def a_new_linear(lm):
    lm.layers[1].mixer.in_proj = copy.deepcopy(lm.layers[1].mixer.in_proj)


def in_place(lm):
    with torch.no_grad():
        lm.layers[1].mixer.in_proj.weight[3, 5] += 1


def swapped(change):
    """The same where torch puts the new tensors into the old Python objects."""
    def run(lm):
        torch.__future__.set_swap_module_params_on_conversion(True)
        try:
            change(lm)
        finally:
            torch.__future__.set_swap_module_params_on_conversion(False)

    return run


def a_training_step(lm):
    for p in lm.parameters():
        p.grad = torch.ones_like(p)
    torch.optim.SGD(lm.parameters(), lr=0.1).step()


CHANGES = [lambda lm: lm.load_state_dict(double(lm)), lambda lm: lm.load_state_dict(double(lm), assign=True), a_new_parameter, a_new_linear,
           in_place, a_training_step, lambda lm: lm.float(), lambda lm: lm.to("meta"), swapped(lambda lm: lm.load_state_dict(double(lm))),
           swapped(lambda lm: lm.float())]


@pytest.mark.parametrize("change", range(len(CHANGES)))
def test_weights_that_changed_are_refused_until_quantised_again(monkeypatch, change):
    lm, rec = small_model(monkeypatch)
    assert taken(lm, rec, monkeypatch)
    CHANGES[change](lm)
    if lm.embedding.weight.dtype == torch.bfloat16 and not lm.embedding.weight.is_meta:
        assert not taken(lm, rec, monkeypatch)
        assert not taken(copy.deepcopy(lm), rec, monkeypatch)
        lm.quantize_linears()
        assert taken(lm, rec, monkeypatch)
    else:
        with pytest.raises(RuntimeError, match="quantize_linears"):
            lm.prefill(torch.zeros(1, 2, dtype=torch.int64))
    lm.quantize_linears(False)
    assert all(layer.mixer._int8 is None and layer.mixer._int8_of is None for layer in lm.layers)


def test_what_leaves_the_weights_as_they_are_is_taken(monkeypatch):
    lm, rec = small_model(monkeypatch)
    lm.eval().train().requires_grad_(False).requires_grad_(True)
    lm.to("cpu").bfloat16().zero_grad()
    with torch.no_grad():
        for layer in lm.layers:  # what is not quantised may change
            layer.norm.weight.mul_(2)
            layer.mixer.x_proj.weight.mul_(2)
    assert taken(lm, rec, monkeypatch)
    held = io.BytesIO()
    torch.save(lm, held)
    held.seek(0)
    for other in (copy.deepcopy(lm), copy.deepcopy(copy.deepcopy(lm)), torch.load(held, weights_only=False)):
        assert taken(other, rec, monkeypatch)
        in_place(lm)
        assert taken(other, rec, monkeypatch) and not taken(lm, rec, monkeypatch)
        in_place(other)
        assert not taken(other, rec, monkeypatch)
        lm.quantize_linears()


def test_inference_tensors_are_taken(monkeypatch):
    Recorder(monkeypatch)
    with torch.inference_mode():
        lm = MambaLM(MambaConfig(d_model=64, n_layer=1, vocab_size=64, dt_rank=8)).bfloat16()
        lm.quantize_linears()
    assert lm.layers[0].mixer.in_proj.weight.is_inference()
    lm.layers[0].mixer._check_int8()


def test_a_weight_that_is_computed_is_not_watched(monkeypatch):
    Recorder(monkeypatch)
    lm = MambaLM(MambaConfig(d_model=64, n_layer=1, vocab_size=64, dt_rank=8)).bfloat16()
    m = lm.layers[0].mixer
    torch.nn.utils.parametrize.register_parametrization(m.in_proj, "weight", torch.nn.Identity())
    lm.quantize_linears()
    m._check_int8()
    with torch.no_grad():
        m.out_proj.weight.mul_(2)
    with pytest.raises(RuntimeError, match="quantize_linears"):
        m._check_int8()
