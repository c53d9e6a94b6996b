"""GPU suite: AdamW8 when parameters or its state change between two steps.  Codes and scales are compared with the update in
64 bits; tolerances of the parameters as in test_gpu_adamw8.py."""
import copy

import numpy as np
import pytest
import torch

from test_gpu_adamw8 import DEV, HP, Oracle, _check, _grads, _pad, _params

pytestmark = pytest.mark.gpu


def _step(opt, params, o, k, dtype):
    _grads(params, 200 + k)
    o.p = np.concatenate([_pad(p) for p in params])
    o.advance(params)
    opt.step()
    _check(opt, params, o, dtype, f"step {k}")


def test_a_model_converted_between_steps():
    """float32 -> bfloat16 -> float32 under one optimizer: the moments go on, every step is the formula's for the type that the
    parameters have then."""
    from medical_image_segmentation_amd.utils.optim import AdamW8
    params = _params([1, 127, 129, 5000, 12289, 0], torch.float32, 31)
    m = torch.nn.Module()
    for i, p in enumerate(params):
        m.register_parameter(f"p{i}", p)
    opt, o = AdamW8(params, **HP), Oracle(params, HP)
    _step(opt, params, o, 0, torch.float32)
    m.bfloat16()
    assert all(p is q for p, q in zip(params, m.parameters())) and params[3].dtype == torch.bfloat16
    _step(opt, params, o, 1, torch.bfloat16)
    _step(opt, params, o, 2, torch.bfloat16)
    m.float()
    _step(opt, params, o, 3, torch.float32)
    for p in params:                                    # another address
        p.data = p.data.clone()
    _step(opt, params, o, 4, torch.float32)
    assert [opt.state[p]["step"] for p in params] == [5] * 6


def test_a_gradient_of_the_type_before():
    from medical_image_segmentation_amd.utils.optim import AdamW8
    p = _params([300], torch.float32, 32)[0]
    opt = AdamW8([p], **HP)
    _grads([p], 1)
    opt.step()
    p.data = p.data.bfloat16()                          # its gradient stays float32
    before = p.detach().clone()
    with pytest.raises(RuntimeError, match="type, device and shape"):
        opt.step()
    assert torch.equal(p, before) and opt.state[p]["step"] == 1


@pytest.mark.parametrize("change", ["channels_last", "fewer", "more", "transposed"])
def test_another_shape_or_memory_order_raises(change):
    from medical_image_segmentation_amd.utils.optim import AdamW8, clip_and_step
    torch.manual_seed(2)
    p = torch.nn.Parameter(torch.randn(8, 6, 3, 3, device=DEV))
    opt = AdamW8([p], **HP)
    p.grad = torch.randn_like(p)
    opt.step()
    kept = p.data
    p.data = {"channels_last": lambda t: t.contiguous(memory_format=torch.channels_last), "fewer": lambda t: t[:4].clone(),
              "more": lambda t: torch.cat([t, t]), "transposed": lambda t: t.transpose(0, 1)}[change](p.data)
    p.grad = None
    p.grad = torch.zeros_like(p)
    before, codes = p.detach().clone(), opt.state[p]["exp_avg"].clone()
    for step in (opt.step, lambda: clip_and_step(opt, [p], 1.0), lambda: opt.moments(p)):
        with pytest.raises(RuntimeError, match="parameter 0 is now"):
            step()
    assert torch.equal(p, before) and torch.equal(opt.state[p]["exp_avg"], codes) and opt.state[p]["step"] == 1
    p.data, p.grad = kept, None                          # back again: it goes on
    p.grad = torch.randn_like(p)
    opt.step()
    assert opt.state[p]["step"] == 2


def _captured():
    from medical_image_segmentation_amd.model.utils.modules import ChannelMLP
    from medical_image_segmentation_amd.utils.graph_step import GraphedTrainStep
    from medical_image_segmentation_amd.utils.optim import AdamW8
    torch.manual_seed(6)
    m = ChannelMLP(16, expansion=2, num_groups=4).to(DEV)
    x = torch.randn(2, 16, 6, 6, device=DEV).contiguous(memory_format=torch.channels_last)
    opt = AdamW8(m.parameters(), **HP)
    step = GraphedTrainStep(m, opt, lambda m, x, y: ((m(x) - y).square().mean(), {}), x, torch.randn_like(x), max_norm=0.5)
    step(x, x)
    return m, opt, step, x


@pytest.mark.parametrize("change", ["type", "address"])
def test_a_captured_step_refuses_parameters_that_it_was_not_captured_for(change):
    """The capture writes to the addresses that the parameters had: those may be another tensor's by now."""
    m, opt, step, x = _captured()
    taken = opt.state[m.narrow.weight]["step"]
    kept = [p.data for p in m.parameters()]              # (alive, so that nothing is written to memory that was given back)
    if change == "type":
        m.bfloat16()
    else:
        m.narrow.weight.data = m.narrow.weight.data.clone()
    with pytest.raises(RuntimeError, match="capture the step again"):
        step(x, x)
    for p, t in zip(m.parameters(), kept):
        p.data = t
    step(x, x)
    assert opt.state[m.narrow.weight]["step"] == taken + 1


def test_a_cleared_state_begins_again():
    from medical_image_segmentation_amd.utils.optim import AdamW8
    params = _params([200, 0, 5000], torch.float32, 41)
    opt, o = AdamW8(params, **HP), Oracle(params, HP)
    for k in range(3):
        _step(opt, params, o, k, torch.float32)
    opt.state.clear()
    assert opt.state_dict()["state"] == {}
    o = Oracle(params, HP)
    for k in range(3, 5):
        _step(opt, params, o, k, torch.float32)
    assert [opt.state[p]["step"] for p in params] == [2, 2, 2]
    saved = opt.state_dict()["state"]                    # what a checkpoint holds is what the step works on
    assert all(torch.equal(saved[i][n], opt.state[p][n]) for i, p in enumerate(params) for n in opt._STATE)
    assert int(saved[2]["exp_avg"].count_nonzero()) > 4000


def test_states_put_in_place_of_others_are_gone_on_from():
    from medical_image_segmentation_amd.utils.optim import AdamW8
    pa, pb = _params([129, 4097], torch.float32, 42), _params([129, 4097], torch.float32, 42)
    oa, ob = AdamW8(pa, **HP), AdamW8(pb, **HP)
    for k in range(3):
        _grads(pa, 300 + k)
        oa.step()
    _grads(pb, 400)
    ob.step()
    with torch.no_grad():
        for p, q in zip(pa, pb):
            q.copy_(p)
    # one tensor at a time, and a whole dict with codes in host memory
    for n in ob._STATE:
        ob.state[pb[0]][n] = oa.state[pa[0]][n].clone()
    ob.state[pb[0]]["step"] = 3
    ob.state[pb[1]] = {n: (t.cpu() if torch.is_tensor(t) else t) for n, t in oa.state[pa[1]].items()}
    _grads(pa, 303)
    _grads(pb, 303)
    oa.step()
    ob.step()
    assert all(torch.equal(p, q) for p, q in zip(pa, pb)) and all(torch.equal(a, b) for a, b in zip(oa.moments(), ob.moments()))
    assert [ob.state[p]["step"] for p in pb] == [4, 4]
    before = pb[0].detach().clone()
    ob.state[pb[0]]["exp_avg"] = torch.zeros(100, device=DEV)
    with pytest.raises(ValueError, match="should be 256 bytes"):
        ob.step()
    assert torch.equal(pb[0], before)


def test_a_captured_step_refuses_a_state_that_it_was_not_captured_for():
    m, opt, step, x = _captured()
    opt.state.clear()
    with pytest.raises(RuntimeError, match="state was replaced after the capture"):
        step(x, x)


def test_a_checkpoint_of_a_channels_last_model():
    """Saved and loaded in its own order it goes on bit for bit; the same model in rows refuses it."""
    from medical_image_segmentation_amd.utils.optim import AdamW8
    torch.manual_seed(8)
    w = torch.randn(8, 6, 3, 3, device=DEV)
    last = w.contiguous(memory_format=torch.channels_last)
    g = [torch.randn_like(w) for _ in range(3)]
    a, b, c = (torch.nn.Parameter(t.clone(memory_format=torch.preserve_format)) for t in (last, last, w))
    oa, ob, oc = (AdamW8([p], **HP) for p in (a, b, c))
    for t in g[:2]:
        a.grad = t.contiguous(memory_format=torch.channels_last)
        oa.step()
    saved = copy.deepcopy(oa.state_dict())
    ob.load_state_dict(saved)
    with torch.no_grad():
        b.copy_(a)
    a.grad, b.grad = g[2].contiguous(memory_format=torch.channels_last), g[2]
    oa.step()
    ob.step()
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(oa.moments(a), ob.moments(b)))
    with pytest.raises(RuntimeError, match="parameter 0 is now"):
        oc.load_state_dict(saved)
    assert not oc.state


@pytest.mark.parametrize("change", [dict(betas=(0.8, 0.99)), dict(eps=1e-6), dict(seed=5)])
def test_a_captured_step_refuses_options_that_its_launches_hold_fast(change):
    """lr and weight_decay are read before every replay; the others are arguments of the captured launches."""
    m, opt, step, x = _captured()
    group = opt.param_groups[0]
    kept, taken = {k: group[k] for k in change}, opt.state[m.narrow.weight]["step"]
    group.update(change)
    with pytest.raises(RuntimeError, match="changed after the capture"):
        step(x, x)
    assert opt.state[m.narrow.weight]["step"] == taken
    group.update(kept, lr=1e-4, weight_decay=0.0)
    step(x, x)
    assert opt.state[m.narrow.weight]["step"] == taken + 1


def test_a_state_that_cannot_be_copied_is_left_as_it_was(monkeypatch):
    """Laying the buffers out again goes through a copy of the old ones; where it fails, the old state is still there."""
    from medical_image_segmentation_amd.utils.optim import AdamW8
    p, q = _params([300], torch.float32, 51)[0], _params([40], torch.float32, 52)[0]
    opt = AdamW8([p], **HP)
    _grads([p], 1)
    opt.step()
    before = [t.clone() for t in opt.moments(p)]
    opt.add_param_group(dict(params=[q]))
    with monkeypatch.context() as m:
        def fails(*args):
            raise RuntimeError("no memory")
        m.setattr(torch, "_foreach_copy_", fails)
        with pytest.raises(RuntimeError, match="no memory"):
            opt.step()
    assert opt.state[p]["step"] == 1 and all(torch.equal(a, b) for a, b in zip(before, opt.moments(p)))
