"""GPU suite: gradients of the 1x1-conv function and of the modules built on it, float32 and bfloat16, against 64-bit formulas;
the block with the 8-bit optimizer under the gradient exchange."""

import pytest
import torch

from operators_ref import act64, group_norm_act64, linear_act64
from test_gpu_norm_linear import ACT_ERR, DEV, H32, _close, _half, _x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pointwise_conv_gradients(dtype, act):
    """All four gradients in nn.Conv2d's layout; tolerances as in _lin_case of test_gpu_norm_linear.py."""
    from medical_image_segmentation_amd import functional as F_
    B, K, N, H, W = 2, 24, 40, 9, 7
    M = B * H * W
    g = torch.Generator().manual_seed(5)
    x, r = _x((B, K, H, W), dtype, 41).requires_grad_(), _x((B, N, H, W), dtype, 42).requires_grad_()
    w = (torch.randn((N, K, 1, 1), generator=g) / K ** 0.5).to(DEV, dtype).requires_grad_()
    b = (torch.randn(N, generator=g) * 0.3).to(DEV).requires_grad_()
    dy = _x((B, N, H, W), dtype, 43)
    y = F_.pointwise_conv_act(x, w, b, act, r)
    got = torch.autograd.grad(y, [x, w, b, r], dy)
    assert [t.shape for t in got] == [x.shape, w.shape, b.shape, r.shape] and [t.dtype for t in got] == [dtype, dtype, b.dtype, dtype]
    rows = lambda t: t.detach().double().permute(0, 2, 3, 1).reshape(M, -1)  # noqa: E731
    xd, wd, bd, dyd = rows(x), w.detach().double()[:, :, 0, 0], b.detach().double(), rows(dy)
    u = (xd @ wd.t() + bd).requires_grad_()
    v = act64(u, act)
    (dz,) = torch.autograd.grad(v, u, dyd)
    h = _half(dtype)
    acc = lambda n: 2 * n ** 0.5 * H32  # noqa: E731
    terms = xd.abs() @ wd.t().abs() + bd.abs()
    smooth = act in ("silu", "gelu")
    u_err = acc(K) * terms
    if act == "relu":
        assert bool((u.detach().abs() > u_err).all())
    want = v.detach() + rows(r)
    _close(y.permute(0, 2, 3, 1).reshape(M, N), want, h * want.abs() + 1.13 * u_err + ACT_ERR * (terms + 1) * smooth
           + 2 * H32 * (v.detach().abs() + rows(r).abs()), "y")
    dz_err = (dyd.abs() * (0.8 * u_err + ACT_ERR * (terms + 1)) + 2 * H32 * dz.abs()) if smooth else 0 * dz
    dz_r = dz_err + h * dz.abs() * (act != "none")
    az, ax, aw = dz.abs(), xd.abs(), wd.abs()
    gx, gw = dz @ wd, dz.t() @ xd
    _close(rows(got[0]), gx, h * gx.abs() + dz_r @ aw + acc(N) * (az @ aw) + 1e-30, "dx")
    _close(got[1][:, :, 0, 0], gw, h * gw.abs() + dz_r.t() @ ax + acc(M) * (az.t() @ ax) + 1e-30, "dweight")
    _close(got[2], dz.sum(0), dz_err.sum(0) + acc(M) * az.sum(0) + 1e-30, "dbias")
    assert torch.equal(got[3], dy)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((2, 32, 12, 10), 8), ((1, 64, 17, 5), 16)])
def test_channel_mlp_gradients(shape, groups, dtype):
    """The block's output and all its gradients against 64-bit formulas that round where the block stores a value in its type:
    the norm's output, the hidden activation, their gradients, dz and the weights.

    A result then differs by its own last rounding, h of the value, and where an intermediate value falls on the other side
    of a rounding border than in 64 bits.  An intermediate is off by at most 2 sqrt(240) 2^-24 of its terms (about ten times
    itself) before it is rounded in steps of 2^-7: one value in 2^-7 / (310 * 2^-24) > 400 moves, by 2 h; in norm 2 h / sqrt(400) =
    0.1 h a stage, four stages at most before any result.  float32: the float32 errors themselves, 5 stages of 2 sqrt(240) h and the
    activation."""
    from medical_image_segmentation_amd.model.utils.modules import ChannelMLP
    B, C, H, W = shape
    torch.manual_seed(7)
    m = ChannelMLP(C, expansion=2, num_groups=groups).to(DEV)
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(torch.randn(p.shape) * (0.3 if p.dim() == 1 else p.shape[1] ** -0.5) + (1.0 if p is m.norm.weight else 0.0))
    x, dy = _x(shape, dtype, 51).requires_grad_(), _x(shape, dtype, 52)
    y = m(x)
    names = [n for n, _ in m.named_parameters()]
    got = dict(zip(["x"] + names, torch.autograd.grad(y, [x] + list(m.parameters()), dy)))
    assert y.dtype == dtype and got["x"].dtype == dtype and all(got[n].dtype == torch.float32 for n in names)

    rnd = lambda t: t.to(dtype).double()  # noqa: E731
    rows = lambda t: t.permute(0, 2, 3, 1).reshape(-1, t.shape[1])  # noqa: E731
    d = {n: p.detach().double() for n, p in m.named_parameters()}
    w1, w2 = rnd(d["widen.weight"][:, :, 0, 0]), rnd(d["narrow.weight"][:, :, 0, 0])
    leaves = [t.requires_grad_() for t in (x.detach().double(), d["norm.weight"], d["norm.bias"])]
    norm = group_norm_act64(leaves[0], groups, leaves[1], leaves[2], 1e-5, "none")
    n = rnd(rows(norm.detach()))
    u = (n @ w1.t() + d["widen.bias"]).requires_grad_()
    hidden = act64(u, "gelu")
    hr = rnd(hidden.detach())
    want_y = linear_act64(hr, w2, d["narrow.bias"], "none", rows(x.detach().double()))
    g = rows(dy.double())
    dh = rnd(g @ w2)
    (dz,) = torch.autograd.grad(hidden, u, dh)
    dn = rnd(rnd(dz) @ w1)
    dx, dgamma, dbeta = torch.autograd.grad(norm, leaves, dn.reshape(B, H, W, C).permute(0, 3, 1, 2))
    want = {"x": dx + dy.double(), "norm.weight": dgamma, "norm.bias": dbeta, "widen.weight": (rnd(dz).t() @ n)[:, :, None, None],
            "widen.bias": dz.sum(0), "narrow.weight": (g.t() @ hr)[:, :, None, None], "narrow.bias": g.sum(0)}
    h = _half(dtype)
    if dtype == torch.float32:
        tol = dict.fromkeys(want, 5 * 31 * H32 + 8 * ACT_ERR)
    else:                    # one rounding (x: that of the norm's gradient and that of the sum), and the values that moved
        tol = {"x": 2 * h, "widen.weight": h, "narrow.weight": h, "norm.weight": 0, "norm.bias": 0, "widen.bias": 0, "narrow.bias": 0}
        tol = {k: v + 0.4 * h for k, v in tol.items()}
    rel = lambda a, e: float((a.double() - e).norm() / e.norm())  # noqa: E731
    assert rel(rows(y.detach()), want_y) < max(h + 0.4 * h, tol["x"] if dtype == torch.float32 else 0)
    for k, e in want.items():
        assert rel(got[k], e) < tol[k], (k, rel(got[k], e) / tol[k])


def test_block_and_optimizer_under_the_gradient_exchange():
    """ChannelMLP with AdamW8 on a communicator of one rank (averaging over one is the identity): gradients that are views of
    the exchange's buckets, three steps bit for bit those without it."""
    import torch.distributed as dist
    from medical_image_segmentation_amd.model.utils.modules import ChannelMLP
    from medical_image_segmentation_amd.parallel import GradSync
    from medical_image_segmentation_amd.utils.optim import AdamW8, clip_and_step
    created = not dist.is_initialized()
    if created:
        err = None
        for port in (29527, 29628, 29729):
            try:
                dist.init_process_group("nccl", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1,
                                        device_id=torch.device(DEV))
                err = None
                break
            except Exception as e:      # noqa: BLE001
                err = e
        if err is not None:
            pytest.skip(f"no process group here: {err}")
    try:
        x = _x((2, 32, 14, 9), torch.bfloat16, 61)
        res = []
        for exchange in (False, True):
            torch.manual_seed(9)
            m = ChannelMLP(32, expansion=2, num_groups=8).to(DEV)
            opt = AdamW8(m.parameters(), lr=1e-2, seed=4)
            sync = GradSync(m, always_reduce=True) if exchange else None
            if sync is not None:
                sync.broadcast_parameters()
            for _ in range(3):
                opt.zero_grad()
                loss = (m(x).float() - 1).square().mean()
                if sync is not None:
                    sync.begin_step()
                loss.backward()
                if sync is not None:
                    sync.finish_step()
                clip_and_step(opt, list(m.parameters()), 0.05)
            torch.cuda.synchronize()
            res.append([p.detach().clone() for p in m.parameters()] + [t.clone() for t in opt.moments()])
            if sync is not None:
                sync.remove()
        assert all(torch.equal(a, b) for a, b in zip(*res))
    finally:
        if created:
            dist.destroy_process_group()
