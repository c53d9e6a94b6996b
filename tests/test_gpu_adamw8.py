"""GPU suite: AdamW with 8-bit moments against the update's formulas in 64 bits (tests/operators_ref.py).

Tolerances.  Codes and scales have to be equal: a moment is formed in 64 bits on both sides and a code differs only where
the two evaluations' last bits decide, which happens for about one value in 2^25 x 2^20.  A parameter is off by its
rounding plus the float32 steps of its update: moments rounded once each, the square root, two products, a sum and a
reciprocal, each at most 2 h32 (the hardware's root and reciprocal are good to one unit)."""
import copy

import numpy as np
import pytest
import torch

import operators_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H32 = 2.0 ** -24
SIZES = [1, 3, 127, 128, 129, 255, 4096, 4097, 10000, 12289, 8, 0, 640]
HP = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=1e-2, seed=0x1234567890ABCDEF)


def _params(sizes, dtype, seed, unaligned=False):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        t = (torch.randn(n, generator=g) * 0.1).to(DEV, dtype)
        if unaligned:
            t = torch.cat([t.new_zeros(1), t])[1:]
        out.append(torch.nn.Parameter(t))
    return out


def _grads(params, seed, scale=1e-2):
    g = torch.Generator().manual_seed(seed)
    for p in params:
        v = torch.randn(p.numel(), generator=g) * scale * torch.exp2(-10 * torch.rand(p.numel(), generator=g))
        p.grad = v.reshape(p.shape).to(DEV, p.dtype)


def _pad(t):
    a = t.detach().double().cpu().numpy().reshape(-1)
    return np.concatenate([a, np.zeros(-len(a) % 128)])


class Oracle:
    """All parameters of an optimizer as one flat padded array, in the order of their offsets."""

    def __init__(self, params, hp):
        self.hp, self.step = hp, 0
        self.p = np.concatenate([_pad(p) for p in params])
        n = len(self.p)
        self.m, self.v = np.zeros(n, np.int64), np.zeros(n, np.int64)
        self.ms, self.vs = np.zeros(n // 128, np.int64), np.zeros(n // 128, np.int64)

    def advance(self, params, max_norm=None):
        self.step += 1
        g = np.concatenate([_pad(p.grad) for p in params])
        norm = float(np.sqrt((g * g).sum()))
        coef = min(1.0, max_norm / (norm + 1e-6)) if max_norm else 1.0
        words = ref.philox(len(g), self.step, self.hp["seed"])
        start = self.p.copy()
        self.p, self.m, self.ms, self.v, self.vs = ref.adamw8_step(
            self.p, g, self.m, self.ms, self.v, self.vs, words, self.hp["lr"], *self.hp["betas"], self.hp["eps"],
            self.hp["weight_decay"], self.step, coef)
        self.moved = np.abs(self.p - start)
        return norm


def _check(opt, params, o, dtype, what):
    names = ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")
    at = 0
    for i, p in enumerate(params):
        n, nb = p.numel(), -(-p.numel() // 128)
        s = opt.state[p]
        want = (o.m[at:at + nb * 128], o.ms[at // 128:at // 128 + nb], o.v[at:at + nb * 128], o.vs[at // 128:at // 128 + nb])
        for k, w in zip(names, want):
            got = s[k].cpu().numpy().astype(np.int64)
            if k == "exp_avg":                                       # (a zero may carry either sign)
                got, w = np.where(got == 128, 0, got), np.where(w == 128, 0, w)
            assert np.array_equal(got, w), f"{what}: tensor {i} ({n} elements): {int((got != w).sum())} of {k} differ"
        h = torch.finfo(dtype).eps / 2
        wantp, moved = o.p[at:at + n], o.moved[at:at + n]
        tol = (h + 2 * H32) * np.abs(wantp) + 16 * H32 * moved + 1e-30
        err = np.abs(p.detach().double().cpu().numpy().reshape(-1) - wantp)
        assert (err <= tol).all(), f"{what}: tensor {i}: parameter off by {err.max()}"
        at += nb * 128


@pytest.mark.parametrize("unaligned", [False, True])
@pytest.mark.parametrize("max_norm", [None, 0.05, 100.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_against_formula(dtype, max_norm, unaligned):
    from medical_image_segmentation_amd.utils.optim import AdamW8, clip_and_step
    params = _params(SIZES, dtype, 1, unaligned)
    opt = AdamW8(params, **HP)
    o = Oracle(params, HP)
    for k in range(4):
        _grads(params, 10 + k)
        before = [p.grad.clone() for p in params]
        norm = o.advance(params, max_norm)
        got = clip_and_step(opt, params, max_norm) if max_norm else opt.step()
        if max_norm:
            assert abs(float(got) - norm) <= 2 * H32 * norm
        _check(opt, params, o, dtype, f"step {k}")
        o.p = np.concatenate([_pad(p) for p in params])              # (parameters go on from what the type holds)
        assert all(torch.equal(p.grad, b) for p, b in zip(params, before))
    m, v = opt.moments()
    assert np.array_equal(m.double().cpu().numpy(), ref.decode(o.m, o.ms, True))
    assert np.array_equal(v.double().cpu().numpy(), ref.decode(o.v, o.vs, False))
    for p in params:
        a, b = opt.moments(p)
        assert a.shape == b.shape == p.shape


def test_mixed_types_groups_and_missing_gradients():
    """Two groups with hyper-parameters of their own, two types, a tensor that gets its first gradient later: every tensor
    follows its own step number; the roundings follow the position in the flat order."""
    from medical_image_segmentation_amd.utils.optim import AdamW8
    a, b = _params([300, 5000], torch.float32, 3), _params([129, 777], torch.bfloat16, 4)
    opt = AdamW8([dict(params=a), dict(params=b, lr=1e-2, weight_decay=0.0)], **HP)
    o = [Oracle([p], {**HP, "lr": lr, "weight_decay": wd}) for p, lr, wd in
         [(p, HP["lr"], HP["weight_decay"]) for p in a] + [(p, 1e-2, 0.0) for p in b]]
    offsets = np.cumsum([0] + [-(-p.numel() // 128) * 128 for p in a + b])
    for k in range(3):
        _grads(a + b, 40 + k)
        if k == 0:
            a[1].grad = None
            frozen = a[1].detach().clone()
        opt.step()
        for i, (p, q) in enumerate(zip(a + b, o)):
            if p.grad is None:
                assert torch.equal(p, frozen) and opt.state[p]["step"] == 0
                continue
            q.step += 1
            g = _pad(p.grad)
            words = ref.philox(int(offsets[-1]), q.step, HP["seed"])[offsets[i]:offsets[i + 1]]
            start = q.p.copy()
            q.p, q.m, q.ms, q.v, q.vs = ref.adamw8_step(q.p, g, q.m, q.ms, q.v, q.vs, words, q.hp["lr"], *HP["betas"],
                                                        HP["eps"], q.hp["weight_decay"], q.step)
            q.moved = np.abs(q.p - start)
            _check(opt, [p], q, p.dtype, f"step {k}, tensor {i}")
            q.p = _pad(p)
    assert [opt.state[p]["step"] for p in a + b] == [3, 2, 3, 3]


def test_extreme_moments():
    """Blocks with zeros, the largest and smallest magnitudes, infinities and NaN, with the second moment never falling to
    zero; a bad block spoils its own 128 elements only."""
    from medical_image_segmentation_amd.utils.optim import AdamW8
    p = _params([128 * 8], torch.float32, 5)[0]
    opt = AdamW8([p], **HP)
    o = Oracle([p], HP)
    g = torch.zeros(8, 128)
    g[1] = torch.exp2(torch.linspace(-40, 0, 128))                    # far wider than a block's range
    g[2] = torch.exp2(torch.linspace(-140, -100, 128))                # squares below float32
    g[3] = 1e15
    g[4, 5] = float("inf")
    g[5, 6] = float("nan")
    g[6, 0] = 1.0                                                     # one value among zeros
    g[7] = torch.linspace(-2, 2, 128) * 1.875
    for k in range(3):
        p.grad = g.reshape(-1).to(DEV)
        o.advance([p])
        opt.step()
        got = {n: opt.state[p][n].cpu().numpy().astype(np.int64) for n in ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")}
        assert np.array_equal(got["exp_avg_scale"], o.ms) and np.array_equal(got["exp_avg_sq_scale"], o.vs)
        bad = np.repeat(o.ms == 255, 128)
        assert list(np.flatnonzero(o.ms == 255)) == [4, 5]
        keep = ~bad
        assert np.array_equal(got["exp_avg"][keep] % 128, o.m[keep] % 128) and np.array_equal(got["exp_avg_sq"][keep], o.v[keep])
        v = opt.moments(p)[1].cpu().numpy()
        assert np.isnan(v[bad]).all() and (v[128:256] > 0).all()
    q = p.detach().cpu().numpy()
    assert np.isfinite(q[:4 * 128]).all() and np.isfinite(q[6 * 128:]).all()


def test_channels_last_parameters_and_gradients():
    """Elements are taken in memory order; a gradient in another order is brought into the parameter's."""
    from medical_image_segmentation_amd.utils.optim import AdamW8
    torch.manual_seed(0)
    w = torch.randn(8, 6, 3, 3, device=DEV)
    a, b = torch.nn.Parameter(w.clone()), torch.nn.Parameter(w.contiguous(memory_format=torch.channels_last))
    c = torch.nn.Parameter(w.contiguous(memory_format=torch.channels_last))
    opts = [AdamW8([p], lr=1e-2) for p in (a, b, c)]
    g = torch.randn_like(w)
    a.grad, b.grad, c.grad = g, g.contiguous(memory_format=torch.channels_last), g
    for o in opts:
        o.step()
    assert torch.equal(b, c) and b.stride() == w.contiguous(memory_format=torch.channels_last).stride()
    assert torch.equal(a, b)                  # (the first update does not depend on the codes)
    assert torch.equal(opts[1].moments(b)[0], opts[2].moments(c)[0])
    assert opts[1].moments(b)[0].stride() == b.stride()


def test_checkpoint_resumes_bit_for_bit():
    from medical_image_segmentation_amd.utils.optim import AdamW8, clip_and_step
    pa = _params(SIZES, torch.float32, 7)
    oa = AdamW8(pa, **HP)
    for k in range(3):
        _grads(pa, 70 + k)
        clip_and_step(oa, pa, 0.5)
    pb = [torch.nn.Parameter(p.detach().clone()) for p in pa]
    ob = AdamW8(pb, lr=9.0)
    ob.load_state_dict(copy.deepcopy(oa.state_dict()))
    for k in range(3):
        _grads(pa, 80 + k)
        for p, q in zip(pa, pb):
            q.grad = p.grad.clone()
        assert torch.equal(clip_and_step(oa, pa, 0.5), clip_and_step(ob, pb, 0.5))
    for p, q in zip(pa, pb):
        assert torch.equal(p, q)
    assert all(torch.equal(a, b) for a, b in zip(oa.moments(), ob.moments()))


def test_added_group_keeps_the_state():
    from medical_image_segmentation_amd.utils.optim import AdamW8
    ps = _params([200, 300], torch.float32, 8)
    opt = AdamW8(ps, **HP)
    _grads(ps, 90)
    opt.step()
    before = [t.clone() for p in ps for t in opt.moments(p)]
    more = _params([77], torch.float32, 9)
    opt.add_param_group(dict(params=more))
    assert all(torch.equal(a, b) for a, b in zip(before, [t for p in ps for t in opt.moments(p)]))
    _grads(ps + more, 91)
    opt.step()
    assert [opt.state[p]["step"] for p in ps + more] == [2, 2, 1]


def test_large_tensor_and_many_tensors():
    """Codes behind the first 2^24 elements and a table of 600 tensors, spot-checked against the formula."""
    from medical_image_segmentation_amd.utils.optim import AdamW8
    n = (1 << 24) + 131
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = AdamW8([p], **HP)
    torch.manual_seed(1)
    p.grad = torch.randn(n, device=DEV)
    opt.step()
    lo = (1 << 24) - 256
    padded = -(-n // 128) * 128
    g = np.concatenate([p.grad[lo:].double().cpu().numpy(), np.zeros(padded - n)])
    words = ref.philox(padded, 1, HP["seed"])[lo:]
    k = len(g)
    z = np.zeros(k, np.int64)
    _, m, ms, v, vs = ref.adamw8_step(np.zeros(k), g, z, z[:k // 128], z, z[:k // 128], words, HP["lr"], *HP["betas"],
                                      HP["eps"], HP["weight_decay"], 1)
    s = opt.state[p]
    assert np.array_equal(s["exp_avg"][lo:].cpu().numpy() % 128, m % 128) and np.array_equal(s["exp_avg_sq"][lo:].cpu().numpy(), v)
    assert np.array_equal(s["exp_avg_scale"][lo // 128:].cpu().numpy(), ms)
    many = _params([1 + (i * 37) % 500 for i in range(600)], torch.float32, 11)
    opt = AdamW8(many, **HP)
    o = Oracle(many, HP)
    _grads(many, 92)
    o.advance(many)
    opt.step()
    _check(opt, many, o, torch.float32, "many")


def test_clip_over_other_tensors_than_are_stepped():
    """A norm over more tensors than the optimizer holds: torch's clipping, then the step."""
    from medical_image_segmentation_amd.utils.optim import AdamW8, clip_and_step
    ps = _params([100, 50], torch.float32, 12)
    _grads(ps, 93, scale=1.0)
    opt = AdamW8(ps[:1], **HP)
    want = torch.sqrt(sum((p.grad.double() ** 2).sum() for p in ps))
    norm = clip_and_step(opt, ps, 0.1)
    assert abs(float(norm) - float(want)) < 1e-5 * float(want)
    assert abs(float(torch.sqrt(sum((p.grad.double() ** 2).sum() for p in ps))) - 0.1) < 1e-4


def test_captured_step_equals_eager():
    """A whole training step with AdamW8 captured and replayed equals eager steps bit for bit, learning-rate changes
    included, and eager steps can follow."""
    from medical_image_segmentation_amd.model.utils.modules import ChannelMLP
    from medical_image_segmentation_amd.utils.graph_step import GraphedTrainStep
    from medical_image_segmentation_amd.utils.optim import AdamW8, clip_and_step
    torch.manual_seed(5)
    ma = ChannelMLP(32, expansion=2, num_groups=4).to(DEV)
    mb = copy.deepcopy(ma)
    loss_of = lambda m, x, y: ((m(x).float() - y).square().mean(), {})  # noqa: E731
    batches = [(torch.randn(2, 32, 8, 8, device=DEV).bfloat16().contiguous(memory_format=torch.channels_last),
                torch.randn(2, 32, 8, 8, device=DEV)) for _ in range(6)]
    oa, ob = AdamW8(ma.parameters(), **HP), AdamW8(mb.parameters(), **HP)

    def eager(k):
        oa.zero_grad()
        loss, _ = loss_of(ma, *batches[k])
        loss.backward()
        return loss.detach(), clip_and_step(oa, list(ma.parameters()), 0.5)

    want = [eager(k) for k in (0, 0, 1, 2)]
    step = GraphedTrainStep(mb, ob, loss_of, *batches[0], max_norm=0.5, warmup=2)
    for k, w in zip((1, 2), want[2:]):
        loss, _, norm = step(*batches[k])
        torch.cuda.synchronize()
        assert torch.equal(loss, w[0]) and torch.equal(norm, w[1])
    for o in (oa, ob):
        o.param_groups[0]["lr"] = 1e-3
    for k in (3, 4):
        w = eager(k)
        loss, _, norm = step(*batches[k])
        torch.cuda.synchronize()
        assert torch.equal(loss, w[0]) and torch.equal(norm, w[1])
    for p, q in zip(ma.parameters(), mb.parameters()):
        assert torch.equal(p, q) and oa.state[p]["step"] == ob.state[q]["step"] == 6
    assert all(torch.equal(a, b) for a, b in zip(oa.moments(), ob.moments()))


def test_eager_step_refuses_to_be_captured():
    from medical_image_segmentation_amd.utils.optim import AdamW8
    ps = _params([64], torch.float32, 14)
    opt = AdamW8(ps, **HP)
    _grads(ps, 94)
    opt.step()
    g = torch.cuda.CUDAGraph()
    keep = torch.zeros(4, device=DEV)
    with torch.cuda.graph(g):
        keep.add_(1)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            opt.step()
    assert opt.state[ps[0]]["step"] == 1
