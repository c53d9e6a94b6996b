"""GPU suite: group norm where float32 alone would lose the result: means far from zero, long sums.

Tolerances: h32 = 2^-24 is one float32 rounding.  The statistics are exact here to far below it, so a normalised value
xh = (x - mean) rstd is off by the rounding of rstd, of x - mean (both sides near each other: one rounding) and of their
product: 4 h32 |xh| with one to spare; u = xh gamma + beta by 6 h32 (|xh gamma| + |beta|) likewise."""
import pytest
import torch

from operators_ref import act64, group_norm_act64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H32 = 2.0 ** -24


def _far(shape, G, m0, seed, steps=64):
    """float32 values that spread over `steps` units in the last place: the grid behind 2^m has the step 2^(m - 23); m between
    `m0` and two more, another one for every group."""
    B, C, H, W = shape
    g = torch.Generator().manual_seed(seed)
    k = torch.randint(0, steps, (B, H, W, C), generator=g).double()
    m = m0 + torch.arange(G).repeat_interleave(C // G) % 3
    x = (2.0 ** m.double()) * (1 + k * 2.0 ** -23)
    assert torch.equal(x.float().double(), x)
    return x.float().to(DEV).permute(0, 3, 1, 2)


def _check(x, G, act, eps, seed):
    """Forward and backward against 64 bits with tolerances relative to xh, not to x."""
    from medical_image_segmentation_amd import functional as F_
    B, C, H, W = x.shape
    g = torch.Generator().manual_seed(seed)
    x = x.requires_grad_()
    w = (torch.randn(C, generator=g) * 0.3 + 1).to(DEV).requires_grad_()
    b = (torch.randn(C, generator=g) * 0.3).to(DEV).requires_grad_()
    dy = torch.randn((B, H, W, C), generator=g).to(DEV).permute(0, 3, 1, 2)
    y = F_.group_norm_act(x, G, w, b, eps=eps, activation=act)
    got = torch.autograd.grad(y, [x, w, b], dy)
    d = [t.detach().double().requires_grad_() for t in (x, w, b)]
    yd = group_norm_act64(d[0], G, d[1], d[2], eps, act)
    want = torch.autograd.grad(yd, d, dy.double())
    n = d[0].detach().reshape(B, G, -1)
    mean = n.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((n - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = ((n - mean) * rstd).reshape(B, C, H, W)
    r = rstd.expand(B, G, n.shape[-1]).reshape(B, C, H, W)
    gam, bet = d[1].detach().abs()[:, None, None], d[2].detach().abs()[:, None, None]
    terms = xh.abs() * gam + bet
    act_err = 2.0 ** -21 * (terms + 1) if act in ("silu", "gelu") else 0 * terms
    u_err = 6 * H32 * terms
    err = (y.double() - yd).abs().detach()
    tol = 2 * H32 * yd.detach().abs() + 1.13 * u_err + act_err
    assert bool((err <= tol).all()), f"y off by {float((err / tol).max()):.3g} times the tolerance"
    # |act'| <= 1.13, |act''| <= 0.8; sums of at most 80 float32 terms in a row, see _gn_case in test_gpu_norm_linear.py
    dyd = dy.double().abs()
    du, du_err = 1.13 * dyd, dyd * (0.8 * u_err * (act in ("silu", "gelu")) + act_err) + 2 * H32 * 1.13 * dyd
    mean_of = lambda t: t.reshape(B, G, -1).mean(-1, keepdim=True).expand(B, G, n.shape[-1]).reshape(B, C, H, W)  # noqa: E731
    t1, t2 = gam * du, gam * du * xh.abs()
    m1 = mean_of(gam * du_err) + 84 * H32 * mean_of(t1)
    m2 = mean_of(gam * du_err * xh.abs()) + 88 * H32 * mean_of(t2)
    dx_tol = r * (gam * du_err + m1 + xh.abs() * m2 + 4 * H32 * xh.abs() * mean_of(t2)
                  + 6 * H32 * (gam * du + mean_of(t1) + xh.abs() * mean_of(t2)))
    s = (0, 2, 3)
    for name, a, e, t in (("dx", got[0], want[0], dx_tol),
                          ("dweight", got[1], want[1], (du_err * xh.abs() + 88 * H32 * du * xh.abs()).sum(s)),
                          ("dbias", got[2], want[2], (du_err + 84 * H32 * du).sum(s))):
        off = (a.double() - e).abs() / (t + 1e-30)
        assert float(off.max()) <= 1, f"{name} off by {float(off.max()):.3g} times the tolerance"


# the resident kernels (the first two) and the streaming ones, with and without vectors inside a group
SHAPES = [((2, 64, 16, 16), 8), ((3, 12, 9, 7), 4), ((1, 48, 200, 210), 6), ((2, 30, 150, 131), 10), ((1, 1001, 9, 9), 7)]


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("shape,G", SHAPES)
def test_spread_far_smaller_than_the_mean(shape, G, act):
    """Values over 64 steps of the float32 grid: a mean rounded to float32 is off by up to half a step, 1/37 of the spread, and
    E[x^2] - mean^2 in 64 bits by 1e-5 of itself."""
    _check(_far(shape, G, 0, shape[1]), G, act, 1e-14, 5)


@pytest.mark.parametrize("C,H,W", [(129, 1500, 1400), (33, 3000, 2500), (8, 6000, 9000)])
def test_bias_gradient_of_long_sums(C, H, W):
    """Every pixel of a channel adds the same du, silu'(beta): dbias is the number of pixels times that.  At most 64 float32
    additions in a row, 8 over the pixel rows of a workgroup, two roundings; one float32 sum of a thread's whole share (500 and
    1000 terms of one size, whose roundings go one way) is 7e-6 off, 110 h32."""
    from medical_image_segmentation_amd import functional as F_
    b = torch.linspace(-1.0, 3.0, C, device=DEV, requires_grad=True)
    grad = []
    for h, w in ((1, 1), (H, W)):
        x = torch.zeros(1, C, h, w, device=DEV, dtype=torch.bfloat16).contiguous(memory_format=torch.channels_last)
        y = F_.group_norm_act(x, 1, None, b, activation="silu")
        grad += torch.autograd.grad(y, [b], torch.ones_like(y))
    one, many = grad[0].double(), grad[1].double()
    err = ((many - H * W * one) / (H * W * one)).abs()
    assert float(err.max()) <= 74 * H32, float(err.max())
