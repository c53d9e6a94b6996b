"""GPU suite: group norm, matrix product and 8-bit AdamW at sizes whose offsets or grids pass 32 bits, and the calls that
their documentation allows and that sharing memory or modes can spoil."""
import numpy as np
import pytest
import torch

import operators_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H16 = 2.0 ** -8          # half a step of bfloat16, relative


def _close(got, want, tol, what):
    """|got - want| <= half a bfloat16 step of the value + tol."""
    err = (got.detach().double() - want.detach()).abs() - H16 * want.detach().abs()
    assert float(err.max()) <= tol, f"{what}: {float(err.max())} above {tol}"


def test_group_norm_more_slabs_than_a_launch_holds():
    """65535 samples of 16384 channels in one pixel: 8.4 million slabs.  Values off by their rounding, plus the float32
    steps: |x| < 7 and rstd < 30 for groups of 8 normals (a variance below 1e-3 has odds of 1e-11 per group), six terms of
    2^-24 each: 7 * 30 * 6 * 2^-24 < 1e-4."""
    from medical_image_segmentation_amd import functional as F_
    B, C, G = 65535, 16384, 2048
    x = torch.randn(B, C, 1, 1, device=DEV, dtype=torch.bfloat16).contiguous(memory_format=torch.channels_last).requires_grad_()
    dy = torch.randn(B, C, 1, 1, device=DEV, dtype=torch.bfloat16)
    w = torch.nn.Parameter(torch.rand(C, device=DEV) + 0.5)
    b = torch.nn.Parameter(torch.randn(C, device=DEV))
    y = F_.group_norm_act(x, G, w, b)
    y.backward(dy)
    dw, db = torch.zeros(C, device=DEV, dtype=torch.float64), torch.zeros(C, device=DEV, dtype=torch.float64)
    size = torch.zeros(C, device=DEV, dtype=torch.float64)
    for i in range(0, B, 8192):
        t = x.detach()[i:i + 8192, :, 0, 0].double().reshape(-1, G, C // G)
        d = dy[i:i + 8192, :, 0, 0].double()
        mean = t.mean(-1, keepdim=True)
        rstd = 1 / torch.sqrt(((t - mean) ** 2).mean(-1, keepdim=True) + 1e-5)
        h = (t - mean) * rstd
        _close(y.detach()[i:i + 8192, :, 0, 0], h.reshape(-1, C) * w.double() + b.double(), 1e-4, f"y from sample {i}")
        u = (d * w.double()).reshape(h.shape)
        want = rstd * (u - u.mean(-1, keepdim=True) - h * (u * h).mean(-1, keepdim=True))
        _close(x.grad[i:i + 8192, :, 0, 0], want.reshape(-1, C), 4e-4, f"dx from sample {i}")
        dw += (d * h.reshape(-1, C)).sum(0)
        db += d.sum(0)
        size += (d.abs() * (1 + h.reshape(-1, C).abs())).sum(0)
    # sums over the samples of float32 values (one rounding each, two for the product with rstd), then one rounding
    assert float(((w.grad - dw).abs() / size).max()) < 6 * 2.0 ** -24
    assert float(((b.grad - db).abs() / size).max()) < 6 * 2.0 ** -24


def test_group_norm_behind_32_bit_offsets():
    """2.4e9 elements.  The sums of the backward are float32 within a thread (below 600 terms here): 600 * 2^-24 < 4e-5 of
    their size."""
    from medical_image_segmentation_amd import functional as F_
    C, G, H, W = 8, 2, 15000, 20000
    n = H * W
    x = torch.randn(1, C, H, W, device=DEV, dtype=torch.bfloat16).contiguous(memory_format=torch.channels_last)
    x = x.requires_grad_()
    dy = (x.detach().abs() + x.detach() / 2).contiguous(memory_format=torch.channels_last)
    w = torch.nn.Parameter(torch.linspace(0.5, 1.5, C, device=DEV))
    b = torch.nn.Parameter(torch.linspace(-1, 1, C, device=DEV))
    y = F_.group_norm_act(x, G, w, b)
    y.backward(dy)
    rows, drows = x.detach().permute(0, 2, 3, 1).reshape(n, C), dy.permute(0, 2, 3, 1).reshape(n, C)
    cut = [slice(i, min(i + (1 << 24), n)) for i in range(0, n, 1 << 24)]
    s1 = sum(rows[c].double().sum(0) for c in cut).reshape(G, -1).sum(1)
    s2 = sum((rows[c].double() ** 2).sum(0) for c in cut).reshape(G, -1).sum(1)
    count = n * C // G
    mean = s1 / count
    rstd = 1 / torch.sqrt(s2 / count - mean * mean + 1e-5)
    mean, rstd = mean.repeat_interleave(C // G), rstd.repeat_interleave(C // G)
    db = sum(drows[c].double().sum(0) for c in cut)
    dw = sum((drows[c].double() * (rows[c].double() - mean) * rstd).sum(0) for c in cut)
    assert float(((b.grad - db) / db).abs().max()) < 1e-4 and float(((w.grad - dw) / dw).abs().max()) < 2e-4
    m1 = ((db * w.double()).reshape(G, -1).sum(1) / count).repeat_interleave(C // G)
    m2 = ((dw * w.double()).reshape(G, -1).sum(1) / count).repeat_interleave(C // G)
    yr, dr = y.detach().permute(0, 2, 3, 1).reshape(n, C), x.grad.permute(0, 2, 3, 1).reshape(n, C)
    for c in (cut[0], slice((1 << 28) - 1000, (1 << 28) + 1000), slice(n - 5000, n)):
        h = (rows[c].double() - mean) * rstd
        _close(yr[c], h * w.double() + b.double(), 1e-5, f"y {c}")
        _close(dr[c], rstd * (drows[c].double() * w.double() - m1 - h * m2), 5e-4, f"dx {c}")


def test_linear_behind_32_bit_offsets():
    """2.6e9 elements of -1, 0, 1: every product and sum is a small integer, so all results but the rounded weight gradient
    are exact."""
    from medical_image_segmentation_amd import functional as F_
    M, K, N = 40_000_003, 64, 64
    draw = lambda *s: torch.randint(-1, 2, s, device=DEV, dtype=torch.int8).to(torch.bfloat16)  # noqa: E731
    x, w, r = draw(M, K).requires_grad_(), draw(N, K).requires_grad_(), draw(M, N)
    b = torch.randint(-1, 2, (N,), device=DEV).float().requires_grad_()
    dy = draw(M, N)
    y = F_.linear_act(x, w, b, "relu", r)
    y.backward(dy)
    dw, db = torch.zeros(N, K, device=DEV, dtype=torch.float64), torch.zeros(N, device=DEV, dtype=torch.float64)
    wf = w.detach().float()
    for i in range(0, M, 1 << 22):
        c = slice(i, min(i + (1 << 22), M))
        u = x.detach()[c].float() @ wf.t() + b.detach()
        assert torch.equal(y.detach()[c].float(), torch.relu(u) + r[c].float()), f"y from row {i}"
        z = dy[c].float() * (u > 0)
        assert torch.equal(x.grad[c].float(), z @ wf), f"dx from row {i}"
        dw += (z.t() @ x.detach()[c].float()).double()
        db += z.double().sum(0)
    assert torch.equal(b.grad.double(), db)
    assert torch.equal(w.grad, dw.to(torch.bfloat16))


def test_adamw8_behind_32_bit_offsets():
    from medical_image_segmentation_amd.utils.optim import AdamW8
    hp = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=1e-2, seed=77)
    n = (1 << 31) + 300
    p = torch.nn.Parameter(torch.ones(n, device=DEV, dtype=torch.bfloat16))
    p.grad = torch.empty_like(p).normal_()
    opt = AdamW8([p], **hp)
    opt.step()
    s, padded = opt.state[p], -(-n // 128) * 128
    for lo, hi in ((0, 1024), ((1 << 31) - 512, padded)):
        k = hi - lo
        g = np.zeros(k)
        g[:min(hi, n) - lo] = p.grad[lo:hi].double().cpu().numpy()
        z = np.zeros(k, np.int64)
        want, m, ms, v, vs = ref.adamw8_step(np.ones(k), g, z, z[:k // 128], z, z[:k // 128],
                                             ref.philox(k, 1, hp["seed"], lo), hp["lr"], *hp["betas"], hp["eps"],
                                             hp["weight_decay"], 1)
        assert np.array_equal(s["exp_avg"][lo:hi].cpu().numpy() % 128, m % 128)
        assert np.array_equal(s["exp_avg_sq"][lo:hi].cpu().numpy(), v)
        assert np.array_equal(s["exp_avg_scale"][lo // 128:hi // 128].cpu().numpy(), ms)
        assert np.array_equal(s["exp_avg_sq_scale"][lo // 128:hi // 128].cpu().numpy(), vs)
        got = p.detach()[lo:hi].double().cpu().numpy()
        want = want[:len(got)]
        assert np.all(np.abs(got - want) <= H16 * np.abs(want) + 1e-6)


def test_adamw8_refuses_parameters_that_share_memory():
    from medical_image_segmentation_amd.utils.optim import AdamW8
    store = torch.zeros(300, device=DEV)
    p, q = torch.nn.Parameter(store[:200]), torch.nn.Parameter(store[199:])
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    with pytest.raises(RuntimeError, match="share memory"):
        AdamW8([p, q]).step()
    q.data = store[200:]
    q.grad = torch.ones_like(q)
    AdamW8([p, q]).step()


def test_inference_mode_and_modules_under_autocast():
    from medical_image_segmentation_amd.model.utils.modules import ChannelMLP
    m = ChannelMLP(32, num_groups=4).to(DEV)
    x = torch.randn(2, 32, 5, 7, device=DEV)
    want = m(x)
    with torch.inference_mode():
        assert torch.equal(m(x), want)
    with torch.no_grad():
        assert torch.equal(m(x), want)
    with torch.autocast("cuda", dtype=torch.bfloat16):       # blocks compute in the type of their input, as DoubleConv does
        assert torch.equal(m(x), want)
        y = m(x.bfloat16())
    assert y.dtype == torch.bfloat16
    # four values rounded on the way (input, norm, hidden, result) and the weights, each by half a step of bfloat16
    assert float((y.double() - want.double()).norm() / want.double().norm()) < 6 * H16


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_activations_at_infinity_and_far_out(act):
    """What the formulas give in float32: a value, an infinity, or NaN where they multiply infinity by zero."""
    from medical_image_segmentation_amd import functional as F_
    v = torch.tensor([float("inf"), float("-inf"), float("nan"), 3e38, -3e38, 100.0, -100.0, 0.0, -0.0], device=DEV)
    got = F_.linear_act(v[:, None], torch.ones(1, 1, device=DEV), None, act)[:, 0].double().cpu()
    want = ref.act64(v.double().cpu(), act).float().double()
    want[2] = float("nan")                    # (the oracle's comparison would take it for negative)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (got, want)
    ok = ~torch.isnan(want)
    assert torch.equal(torch.isinf(got[ok]), torch.isinf(want[ok]))
    fine = ok & ~torch.isinf(want)
    assert bool(((got - want)[fine].abs() <= 4 * 2.0 ** -24 * want[fine].abs() + 1e-37).all()), (got, want)


def test_the_same_tensor_in_every_place():
    """x as its own weight and residual: the gradients of the three uses add up."""
    from medical_image_segmentation_amd import functional as F_
    t = torch.randn(48, 48, device=DEV, requires_grad=True)
    F_.linear_act(t, t, None, "silu", t).backward(torch.ones(48, 48, device=DEV))
    r = t.detach().double().requires_grad_()
    ref.linear_act64(r, r, None, "silu", r).backward(torch.ones(48, 48, device=DEV, dtype=torch.float64))
    # 96 terms of products of |t| < 5 per element, each off by at most 48 roundings of the sum: 1e-5 of the whole
    assert float((t.grad - r.grad).norm() / r.grad.norm()) < 1e-5


@pytest.mark.parametrize("op", ["group_norm_act", "linear_act"])
def test_captured_backward_refuses_leaves_of_a_living_eager_graph(op):
    """The gradient node of a leaf that an eager graph on the default stream keeps alive cannot take part in a capture."""
    from medical_image_segmentation_amd import functional as F_
    w = torch.ones(32, device=DEV, requires_grad=True)
    m = torch.randn(32, 32, device=DEV, requires_grad=True)
    x = torch.randn(2, 32, 6, 6, device=DEV).contiguous(memory_format=torch.channels_last)
    leaf = w if op == "group_norm_act" else m
    run = lambda: F_.group_norm_act(x, 4, w) if op == "group_norm_act" else F_.pointwise_conv_act(x, m)  # noqa: E731
    alive = run()
    (want,) = torch.autograd.grad(alive, [leaf], torch.ones_like(alive), retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph of the same leaf is alive"):
        with torch.cuda.graph(graph):
            y = run()
            torch.autograd.grad(y, [leaf], torch.ones_like(y))
    del alive, y
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
        (got,) = torch.autograd.grad(y, [leaf], torch.ones_like(y))
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_adamw8_loads_a_state_from_the_host_and_keeps_nothing_of_it():
    import io
    from medical_image_segmentation_amd.utils.optim import AdamW8

    def make():
        g = torch.Generator().manual_seed(5)
        ps = [torch.nn.Parameter((torch.randn(n, generator=g) * 0.1).to(DEV)) for n in (300, 0, 128, 4097)]
        for p in ps:
            p.grad = torch.full_like(p, 1e-2)
        return ps, AdamW8(ps, lr=1e-2, seed=9)

    pa, oa = make()
    oa.step()
    file = io.BytesIO()
    torch.save(oa.state_dict(), file)
    file.seek(0)
    pb, ob = make()
    with torch.no_grad():
        for p, q in zip(pb, pa):
            p.copy_(q)
    state = torch.load(file, map_location="cpu", weights_only=True)
    state["state"][0]["exp_avg"][300:] = 77              # codes behind the last element mean nothing
    ob.load_state_dict(state)
    pc, oc = make()
    with torch.no_grad():
        for p, q in zip(pc, pa):
            p.copy_(q)
    oc.load_state_dict(oa.state_dict())                  # the live buffers of another optimizer
    oa.step(), ob.step(), oc.step()
    for a, b, c in zip(pa, pb, pc):
        assert torch.equal(a, b) and torch.equal(a, c)
    for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
        for a, b, c in zip(pa, pb, pc):
            assert torch.equal(oa.state[a][k], ob.state[b][k]) and torch.equal(oa.state[a][k], oc.state[c][k])
    assert [oc.state[p]["step"] for p in pc] == [2, 2, 2, 2]


def test_two_threads_on_two_streams():
    """The same block trained from two threads at once, each with its own stream and optimizer: the results of one alone."""
    import threading
    from medical_image_segmentation_amd.model.utils.modules import ChannelMLP
    from medical_image_segmentation_amd.utils.optim import AdamW8, clip_and_step

    def train(seed, out):
        g = torch.Generator().manual_seed(seed)
        m = ChannelMLP(32, num_groups=4)
        with torch.no_grad():
            for p in m.parameters():
                p.copy_(torch.randn(p.shape, generator=g) * 0.1)
        xs = [torch.randn(2, 32, 24, 20 + seed, generator=g) for _ in range(5)]
        with torch.cuda.stream(torch.cuda.Stream()):
            m.to(DEV)
            opt = AdamW8(m.parameters(), lr=1e-2, seed=seed)
            for x in xs:
                opt.zero_grad()
                m(x.to(DEV)).square().mean().backward()
                clip_and_step(opt, m.parameters(), 0.5)
            torch.cuda.current_stream().synchronize()
        out[seed] = [p.detach().clone() for p in m.parameters()]
        torch.cuda.synchronize()

    alone, both = {}, {}
    for s in (1, 2):
        train(s, alone)
    threads = [threading.Thread(target=train, args=(s, both)) for s in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for s in (1, 2):
        assert all(torch.equal(a, b) for a, b in zip(alone[s], both[s]))
