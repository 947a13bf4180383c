"""The 8-bit linear path without a GPU: which calls in place are taken."""
import pytest
import torch

from mamba_tp_lite_b200 import int8 as Q
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
