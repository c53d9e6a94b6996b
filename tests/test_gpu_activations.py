"""GPU suite: the activations of the matrix product and the group norm in float32, relative to the value itself.

Tolerance of Phi(-|u|) = t P(t) e^(-u^2/2), in h = 2^-24: the fit 1.5e-7 < 3 h; t by a rounded sum and a reciprocal good to 2 h, each
passed on at most in full: 3 h; eight roundings of the polynomial, whose terms are at most 0.9 in sum against a value of 0.5 and
shrink with t: 8 h; two products 2 h; 2^x 2 h; its argument 0.7213 u^2 with a constant and two products rounded, times ln 2:
3 * 0.5 u^2 h = 1.5 u^2 h.  With the value's last rounding: (19 + 1.5 u^2) h."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H32 = 2.0 ** -24


def _gelu(v):
    """v through a product with one column and one row of 1, and the derivative there."""
    from medical_image_segmentation_amd import functional as F_
    x, w = v[:, None].clone().requires_grad_(), torch.ones(1, 1, device=DEV)
    y = F_.linear_act(x, w, None, "gelu")
    return y.detach()[:, 0].double(), torch.autograd.grad(y, x, torch.ones_like(y))[0][:, 0].double()


def test_gelu_relative_to_itself():
    """Down to -12, where the value is 2e-32.  A fit that is good to 1.5e-7 of 1 alone would be 5e-5 off at -3."""
    v = torch.linspace(-12, 12, 400_001, device=DEV)
    y, dy = _gelu(v)
    u = v.double()
    q = 0.5 * torch.special.erfc(u.abs() / math.sqrt(2.0))           # Phi(-|u|)
    rel = (19 + 1.5 * u * u) * H32
    want = torch.where(u < 0, u * q, u - u * q)
    err = (y - want).abs() / ((u * q).abs() * rel + H32 * want.abs() + 1e-45)
    assert float(err.max()) <= 1, (float(err.max()), float(v[err.argmax()]))
    # slope Phi(u) + u phi(u): both terms with that relative error, and the rounding of the constant and the sum
    phi = u * torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi)
    slope = torch.where(u < 0, q, 1 - q) + phi
    err = (dy - slope).abs() / ((q + phi.abs()) * rel + 2 * H32 * slope.abs() + H32 * (u >= 0))
    assert float(err.max()) <= 1, (float(err.max()), float(v[err.argmax()]))


def test_gelu_far_out():
    """Beyond float32's smallest numbers the value is zero or the input itself, and stays finite."""
    v = torch.tensor([-3e38, -1e4, -60.0, -14.5, 14.5, 60.0, 1e4, 3e38], device=DEV)
    y, dy = _gelu(v)
    assert bool((y[:4].abs() <= 1e-37).all()) and torch.equal(y[4:], v[4:].double())
    assert bool((dy[:4].abs() <= 1e-37).all()) and torch.equal(dy[4:], torch.ones_like(dy[4:]))
