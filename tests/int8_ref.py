"""The 8-bit linear path from its definitions in 64 bits (torch on any device), for the tests.

Bounds used with it, u = 2^-24 the half step of fp32:
  scale   fp32(max(a, 1e-8) / 127): within u of the 64-bit quotient, relative.  The norm's a is itself computed in 64 bits
          over n values in an order of its own: relative difference below (n + 10) 2^-53 < 2^-35 for n <= 131071.
  codes   the nearest multiple of the scale: |y / scale - code| <= 1/2, plus what the 64-bit y may be off, 127 * 2^-35.
  linear  the sum is exact, then fp32 operations in a given order, each correctly rounded: equal bits."""
import torch

U = 2.0 ** -24
SLACK = 127 * 2.0 ** -35


def check_rows(codes, scale, y):
    """codes and scale of 64-bit rows y [rows, C], with NaN rows where y is not finite."""
    assert codes.dtype == torch.int8 and scale.dtype == torch.float32
    y = y.double()
    bad = ~torch.isfinite(y).all(-1)
    assert torch.equal(torch.isnan(scale), bad), "NaN scales"
    assert (codes[bad] == 0).all(), "codes of rows that are not finite"
    y, codes, scale = y[~bad], codes[~bad].double(), scale[~bad].double()
    want = y.abs().amax(-1).clamp(min=1e-8) / 127
    assert ((scale - want).abs() <= want * (U + 2.0 ** -35)).all(), "scale"
    assert codes.abs().amax() <= 127 if codes.numel() else True
    off = (y / scale.unsqueeze(-1) - codes).abs()
    # the largest value's quotient may pass 127 by the scale's rounding
    assert (off <= 0.5 + SLACK).all(), f"codes: {off.max().item()}"
    # its code is +-127 but where the floor of the scale counts
    floor = y.abs().amax(-1) < 1e-8
    assert (codes.abs().amax(-1)[~floor] == 127).all()


def add(x, residual):
    return (x.float() + residual.float()).to(residual.dtype)


def norm(h, weight, eps):
    h = h.double()
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + float(torch.tensor(eps, dtype=torch.float32))) * weight.double()


def sums(a, w):
    """Exact sums of int8 products: whole numbers below 2^53 in 64-bit floating point."""
    return a.double() @ w.double().T


def linear(a, a_scale, w, w_scale, bias, dtype):
    y = sums(a, w).float() * a_scale.unsqueeze(-1) * w_scale  # the sum to fp32, then product by product
    if bias is not None:
        y = y + bias.float()
    return y.to(dtype)
