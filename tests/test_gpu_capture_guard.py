"""GPU suite: a captured backward pass of the group-norm and matrix-product operators raises while an eager graph of a leaf that
it reaches is alive, however the leaf gets into the operator; the capture works once that graph is gone.  (Without the refusal
the process would end at the end of the capture: the refusal comes first, while the pass still runs.)"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _cases():
    """name -> (the leaf, a call that uses it)"""
    from medical_image_segmentation_amd import functional as F_
    from medical_image_segmentation_amd.model.utils.modules import ChannelMLP, PointwiseConvAct
    torch.manual_seed(3)
    x = torch.randn(12, 16, device=DEV)
    act = torch.randn(2, 16, 5, 5, device=DEV).contiguous(memory_format=torch.channels_last)
    leaf = lambda *s: torch.randn(s, device=DEV).requires_grad_()  # noqa: E731
    w, r, t, b, v = leaf(8, 16), leaf(12, 8), leaf(16, 8), leaf(16), leaf(8, 16, 1, 1)
    conv, mlp = PointwiseConvAct(16, 8, activation="silu").to(DEV), ChannelMLP(16, expansion=2, num_groups=4).to(DEV)
    return {
        "residual": (r, lambda: F_.linear_act(x, w, None, "gelu", r)),
        "transposed weight": (t, lambda: F_.linear_act(x, t.t(), None, "gelu")),
        "every second bias": (b, lambda: F_.linear_act(x, w.detach(), b[::2], "none")),
        "bias of another stride": (b, lambda: F_.group_norm_act(act, 4, None, b.as_strided((16,), (1,)).flip(0), activation="silu")),
        "4-d weight": (v, lambda: F_.pointwise_conv_act(act, v, None, "relu")),
        "weight of a module": (conv.weight, lambda: conv(act)),
        "weight of a module, cast": (conv.weight, lambda: conv(act.bfloat16())),
        "behind another operator": (mlp.norm.weight, lambda: mlp(act)),
        "input through torch": (b, lambda: F_.group_norm_act((act * b[:, None, None]), 4, activation="gelu")),
    }


NAMES = ["residual", "transposed weight", "every second bias", "bias of another stride", "4-d weight", "weight of a module",
         "weight of a module, cast", "behind another operator", "input through torch"]


@pytest.mark.parametrize("name", NAMES)
def test_a_living_eager_graph_is_refused(name):
    leaf, run = _cases()[name]
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


def test_leaves_that_the_pass_does_not_reach_are_no_obstacle():
    from medical_image_segmentation_amd import functional as F_
    torch.manual_seed(4)
    x, w = torch.randn(12, 16, device=DEV, requires_grad=True), torch.randn(8, 16, device=DEV, requires_grad=True)
    alive = w * 2                                    # an eager graph of w on the default stream
    y = F_.linear_act(x, w, None, "silu")
    (want,) = torch.autograd.grad(y, [x], torch.ones_like(y))
    del y
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = F_.linear_act(x, w, None, "silu")
        (got,) = torch.autograd.grad(y, [x], torch.ones_like(y))
    for _ in range(2):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert alive.requires_grad
