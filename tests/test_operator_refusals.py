"""CPU suite: what the group-norm, matrix-product and 8-bit optimizer entry points refuse, before any launch."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(4096)        # a pointer value that the argument checks accept and nothing reads


def _refused(name, *args, match=None):
    from medical_image_segmentation_amd import _lib
    with pytest.raises(RuntimeError, match=match):
        _lib.call(name, *args)


def test_group_norm_c_entry():
    fwd = lambda *, x=P, dtype=0, B=1, HW=4, C=8, G=2, eps=1e-5, act=0, y=P, stats=P, ws=P: (  # noqa: E731
        x, dtype, B, HW, C, G, None, None, eps, act, y, stats, ws, None)
    for bad in (dict(x=None), dict(dtype=2), dict(B=0), dict(HW=0), dict(C=0), dict(G=3), dict(G=0), dict(eps=-1.0),
                dict(act=4), dict(act=-1), dict(y=None), dict(stats=None), dict(ws=None), dict(C=70000, G=1), dict(B=70000),
                dict(x=ctypes.c_void_p(4098)), dict(stats=ctypes.c_void_p(4104)), dict(eps=float("nan"))):
        _refused("mis_group_norm_act_fwd", *fwd(**bad), match="group_norm_act_fwd")
    bwd = lambda *, x=P, dy=P, dtype=1, B=1, HW=4, C=8, G=2, stats=P, act=0, ws=P: (  # noqa: E731
        x, dy, dtype, B, HW, C, G, None, None, stats, act, None, None, None, ws, None)
    for bad in (dict(x=None), dict(dy=None), dict(dtype=-1), dict(G=5), dict(stats=None), dict(act=9), dict(ws=None),
                dict(dy=ctypes.c_void_p(4097))):
        _refused("mis_group_norm_act_bwd", *bwd(**bad), match="group_norm_act_bwd")


def test_linear_c_entry():
    fwd = lambda *, x=P, ldx=8, w=P, r=None, ldr=0, dtype=0, M=4, N=8, K=8, act=0, y=P, ws=P: (  # noqa: E731
        x, ldx, w, None, r, ldr, dtype, M, N, K, act, y, ws, None)
    for bad in (dict(x=None), dict(w=None), dict(y=None), dict(ldx=7), dict(r=P, ldr=7), dict(dtype=3), dict(M=0), dict(N=0),
                dict(K=0), dict(M=1 << 31), dict(act=5), dict(x=ctypes.c_void_p(4098)), dict(K=1 << 21, ldx=1 << 21), dict(ws=None)):
        _refused("mis_linear_act_fwd", *fwd(**bad), match="linear_act_fwd")
    bwd = lambda *, x=P, ldx=8, dy=P, ldd=8, M=4, ws=P, act=0: (  # noqa: E731
        x, ldx, P, None, dy, ldd, 1, M, 8, 8, act, None, None, None, ws, None)
    for bad in (dict(x=None), dict(dy=None), dict(ldx=1), dict(ldd=1), dict(M=-1), dict(ws=None), dict(act=4),
                dict(ws=ctypes.c_void_p(4104))):
        _refused("mis_linear_act_bwd", *bwd(**bad), match="linear_act_bwd")


def test_adamw8_c_entry():
    _refused("mis_adamw8_sqsum", None, P, 1, 1, P, None, match="adamw8_sqsum")
    _refused("mis_adamw8_sqsum", P, P, 0, 1, P, None, match="adamw8_sqsum")
    step = lambda *, descs=P, n=1, c0=0, c1=1, nc=1, m=P, b1=0.9, b2=0.99, t=1: (  # noqa: E731
        descs, P, n, c0, c1, nc, m, P, P, P, None, 0.0, 1e-3, b1, b2, 1e-8, 0.0, t, 0, None, None, None)
    for bad in (dict(descs=None), dict(n=0), dict(c0=1), dict(c1=2), dict(c0=-1), dict(m=None), dict(b1=1.0), dict(b2=-0.1),
                dict(t=0), dict(m=ctypes.c_void_p(4097))):
        _refused("mis_adamw8_step", *step(**bad), match="adamw8_step")
    _refused("mis_adamw8_moments", P, P, P, P, 0, P, P, None, match="adamw8_moments")
    _refused("mis_adamw8_moments", P, P, P, P, 1, ctypes.c_void_p(4104), P, None, match="adamw8_moments")
    _refused("mis_adamw8_step_constants", 1e-3, 0.9, 0.99, 0.0, 0, P, match="adamw8_step_constants")


def test_functional_refusals():
    from medical_image_segmentation_amd import functional as F_
    x4, x2, w2 = torch.zeros(1, 8, 4, 4), torch.zeros(3, 8), torch.zeros(5, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        F_.group_norm_act(x4, 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        F_.linear_act(x2, w2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        F_.pointwise_conv_act(x4, w2)
    with pytest.raises(ValueError, match="unknown activation"):
        F_.linear_act(x2, w2, activation="tanh")
    with pytest.raises(ValueError, match="unknown activation"):
        F_.group_norm_act(x4, 2, activation=None)
    from medical_image_segmentation_amd.model.utils.modules import GroupNormAct, PointwiseConvAct
    with pytest.raises(ValueError, match="unknown activation"):
        GroupNormAct(2, 8, activation="swish")
    with pytest.raises(ValueError, match="unknown activation"):
        PointwiseConvAct(2, 8, activation="swish")


def test_adamw8_refusals():
    from medical_image_segmentation_amd.utils.optim import AdamW8, clip_and_step
    p = torch.nn.Parameter(torch.zeros(4))
    for bad in (dict(lr=-1.0), dict(eps=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(weight_decay=-1.0),
                dict(seed=-1), dict(seed=1 << 64)):
        with pytest.raises(ValueError):
            AdamW8([p], **bad)
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        AdamW8([torch.nn.Parameter(torch.zeros(4, dtype=torch.float64))])
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        AdamW8([torch.nn.Parameter(torch.zeros(4).half())])
    opt = AdamW8([p])
    opt.step()                                    # no gradient: nothing to do
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="on one GPU"):
        opt.step()
    with pytest.raises(RuntimeError, match="on one GPU"):
        clip_and_step(opt, [p], 1.0)
    codes = dict(exp_avg=torch.zeros(128, dtype=torch.uint8), exp_avg_scale=torch.zeros(1, dtype=torch.uint8),
                 exp_avg_sq=torch.zeros(128, dtype=torch.uint8), exp_avg_sq_scale=torch.zeros(1, dtype=torch.uint8), step=3)
    groups = opt.state_dict()["param_groups"]
    with pytest.raises(ValueError, match="has no exp_avg_scale"):
        opt.load_state_dict({"state": {0: {"step": 1, "exp_avg": codes["exp_avg"]}}, "param_groups": groups})
    with pytest.raises(ValueError, match="should be 128 bytes"):
        opt.load_state_dict({"state": {0: {**codes, "exp_avg": torch.zeros(4, dtype=torch.uint8)}}, "param_groups": groups})
    with pytest.raises(ValueError, match="should be 1 bytes"):
        opt.load_state_dict({"state": {0: {**codes, "exp_avg_scale": torch.zeros(1)}}, "param_groups": groups})
    opt.load_state_dict({"state": {0: codes}, "param_groups": groups})
    assert opt.state[p]["step"] == 3 and opt.state[p]["exp_avg"].dtype == torch.uint8


def test_adamw8_takes_a_parameter_once():
    from medical_image_segmentation_amd.utils.optim import AdamW8
    p, q = torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(4))
    with pytest.warns(UserWarning), pytest.raises(ValueError, match="takes each parameter once"):
        AdamW8([p, q, p])
    opt = AdamW8([p])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[p]))
    assert len(opt.param_groups) == 1


def test_grids_that_no_launch_holds():
    """2^30 rows of one column would need 2^24 tiles of 256 threads; a launch holds below 2^32 threads."""
    from medical_image_segmentation_amd._lib import query
    assert query("mis_linear_act_fwd_workspace_bytes", 1, (1 << 30) - 1, 1, 1) == 0
    assert query("mis_linear_act_fwd_workspace_bytes", 1, ((1 << 24) - 8) * 64, 1, 1) > 0
    _refused("mis_linear_act_fwd", P, 1, P, None, None, 1, 1, (1 << 30) - 1, 1, 1, 0, P, P, None, match="bad dtype or sizes")
