"""CPU suite: what AdamW8 keeps from one step to the next, and when it may not be used any more."""
import pytest
import torch


def _params(*shapes):
    g = torch.Generator().manual_seed(1)
    return [torch.nn.Parameter(torch.randn(s, generator=g)) for s in shapes]


def _converted():
    """(what is done, whether the moments' codes still fit) for a parameter [6, 4, 3, 3] that stays the same object."""
    def typed(p):
        p.data = p.data.bfloat16()

    def order(p):
        p.data = p.data.contiguous(memory_format=torch.channels_last)

    def fewer(p):
        p.data = p.data[:3].contiguous()

    def shape(p):
        p.data = p.data.reshape(4, 6, 3, 3)

    def transposed(p):
        p.data = p.data.transpose(0, 1)

    return [(typed, True), (order, False), (fewer, False), (shape, False), (transposed, False)]


@pytest.mark.parametrize("change,fits", _converted())
def test_tables_of_a_converted_parameter_are_not_used_again(change, fits):
    """The kernels take a tensor's address, length and type from these tables: with those of another type or length they would
    read and write behind its end."""
    from medical_image_segmentation_amd.utils.optim import _Plan8, _check_layout, _layout
    params = _params((5,), (6, 4, 3, 3), (0,))
    plan = _Plan8(params, torch.device("cpu"))
    assert plan.matches(params)
    params[1].data = params[1].data.clone()                 # another address alone: looked up at every step
    assert plan.matches(params)
    state = {"layout": _layout(params[1])}
    change(params[1])
    assert not plan.matches(params)
    if fits:
        _check_layout(1, params[1], state)
    else:
        with pytest.raises(RuntimeError, match="parameter 1 is now"):
            _check_layout(1, params[1], state)


def test_a_module_converted_in_place():
    from medical_image_segmentation_amd.utils.optim import _Plan8
    m = torch.nn.Conv2d(4, 6, 3)
    params = list(m.parameters())
    plan = _Plan8(params, torch.device("cpu"))
    m.bfloat16()
    assert all(a is b for a, b in zip(params, m.parameters())) and not plan.matches(params)
    m.float()
    assert plan.matches(params)
    m.to(memory_format=torch.channels_last)
    assert not plan.matches(params)
    m.half()
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        _Plan8(params, torch.device("cpu"))


def test_layouts_that_are_the_same_memory_order():
    from medical_image_segmentation_amd.utils.optim import _layout
    w = torch.zeros(8, 3, 1, 1)
    assert _layout(w) == _layout(w.contiguous(memory_format=torch.channels_last)) == ((8, 3, 1, 1), (0, 1))
    w = torch.zeros(8, 3, 2, 2)
    assert _layout(w) != _layout(w.contiguous(memory_format=torch.channels_last))
    assert _layout(torch.zeros(4, 0, 3)) == _layout(torch.zeros(3, 0, 4).transpose(0, 2)) == ((4, 0, 3), ())
    assert _layout(torch.zeros(())) == ((), ())


def test_gradients_of_another_size_are_not_taken():
    """The kernels read as many elements of a gradient as its parameter has."""
    from medical_image_segmentation_amd import functional as F_
    from medical_image_segmentation_amd.utils.optim import _Plan8, _Table8
    p, q = _params((4,), (7,))
    p.grad, q.grad = torch.ones(4), torch.ones(7)
    assert F_._native().step_pointers([p, q], -1) == [p.data_ptr(), p.grad.data_ptr(), q.data_ptr(), q.grad.data_ptr()]
    q.data = torch.zeros(9)
    assert q.grad.numel() == 7 and F_._native().step_pointers([p, q], -1) == []
    plan = _Plan8([p, q], torch.device("cpu"))
    plan.device = type("Host", (), {"index": -1})        # (what a host tensor gives for its device)
    table = object.__new__(_Table8)
    table.plan, table.order, table.plain, table.dtypes = plan, [p, q], [True, True], [torch.float32] * 2
    with pytest.raises(RuntimeError, match="type, device and shape"):
        table.addresses()


def test_a_cleared_or_replaced_state_is_noticed():
    from medical_image_segmentation_amd.utils.optim import AdamW8, _Plan8
    params = _params((5,), (300,), (0,))
    opt = AdamW8(params)
    plan = _Plan8(params, torch.device("cpu"))
    codes = lambda n: {k: torch.zeros(n if k.endswith("_scale") else 128 * n, dtype=torch.uint8)  # noqa: E731
                       for k in AdamW8._STATE}
    for p, n in zip(params, (1, 3, 0)):
        opt.state[p] = {"step": 1, **codes(n)}
    plan.keep(opt.state)
    assert plan.holds(opt.state)
    opt.state[params[0]]["step"] = 7                       # (numbers are looked up at every step)
    assert plan.holds(opt.state)
    kept = dict(opt.state)
    for change in (lambda: opt.state.clear(), lambda: opt.state.pop(params[1]),
                   lambda: opt.state.__setitem__(params[0], dict(kept[params[0]])),
                   lambda: opt.state[params[1]].__setitem__("exp_avg_sq", torch.zeros(384, dtype=torch.uint8)),
                   lambda: opt.state[params[1]].pop("exp_avg_scale"), lambda: opt.state.__setitem__(params[2], None)):
        change()
        assert not plan.holds(opt.state)
        opt.state.clear()
        for p, n in zip(params, (1, 3, 0)):
            opt.state[p] = {"step": 1, **codes(n)}
        plan.keep(opt.state)


def test_what_is_put_into_the_state_is_checked():
    from medical_image_segmentation_amd.utils.optim import AdamW8, _check_codes
    z = lambda n, dtype=torch.uint8: torch.zeros(n, dtype=dtype)  # noqa: E731
    good = dict(exp_avg=z(384), exp_avg_scale=z(3), exp_avg_sq=z(384), exp_avg_sq_scale=z(3))
    assert _check_codes(0, 300, good) and not _check_codes(0, 300, {"step": 3})
    for k in AdamW8._STATE:
        with pytest.raises(ValueError, match=f"has no {k}"):
            _check_codes(0, 300, {j: t for j, t in good.items() if j != k})
        with pytest.raises(ValueError, match="bytes, got"):
            _check_codes(0, 300, {**good, k: good[k].float()})
        with pytest.raises(ValueError, match="bytes, got"):
            _check_codes(0, 300, {**good, k: good[k][:-1]})


def _saved(p, step=3):
    """A state dict of AdamW8 for one parameter, as a run that held it in this memory order leaves it."""
    from medical_image_segmentation_amd.utils.optim import AdamW8, _layout
    opt, n = AdamW8([p]), -(-p.numel() // 128)
    codes = lambda k, seed: torch.randint(0, 255, (k,), generator=torch.Generator().manual_seed(seed), dtype=torch.uint8)  # noqa: E731
    opt.state[p] = dict(step=step, exp_avg=codes(128 * n, 1), exp_avg_scale=codes(n, 2), exp_avg_sq=codes(128 * n, 3),
                        exp_avg_sq_scale=codes(n, 4), layout=_layout(p))
    return opt.state_dict()


def test_a_checkpoint_is_loaded_into_its_own_memory_order_alone():
    """The codes lie in the order of the parameter's memory: in another one every moment would be another element's."""
    import io
    from medical_image_segmentation_amd.utils.optim import AdamW8
    torch.manual_seed(0)
    rows = torch.randn(6, 4, 3, 3)
    last = rows.contiguous(memory_format=torch.channels_last)
    for made in (rows, last):
        file = io.BytesIO()
        torch.save(_saved(torch.nn.Parameter(made.clone(memory_format=torch.preserve_format))), file)
        file.seek(0)
        state = torch.load(file, weights_only=True)
        for to in (rows, last):
            p = torch.nn.Parameter(to.clone(memory_format=torch.preserve_format))
            opt = AdamW8([p], lr=0.5)
            if made is to:
                opt.load_state_dict(state)
                assert torch.equal(opt.state[p]["exp_avg"], state["state"][0]["exp_avg"]) and opt.state[p]["step"] == 3
                assert opt.param_groups[0]["lr"] == 1e-3
            else:
                with pytest.raises(RuntimeError, match="parameter 0 is now"):
                    opt.load_state_dict(state)
                assert not opt.state and opt.param_groups[0]["lr"] == 0.5         # nothing was replaced
        del state["state"][0]["layout"]                          # no record: row-major
        opt = AdamW8([torch.nn.Parameter(rows.clone())])
        opt.load_state_dict(state)
        opt = AdamW8([torch.nn.Parameter(last.clone(memory_format=torch.preserve_format))])
        with pytest.raises(RuntimeError, match="by falling stride"):
            opt.load_state_dict(state)
    with pytest.raises(RuntimeError, match="parameter 0 is now"):
        AdamW8([torch.nn.Parameter(rows.reshape(4, 6, 3, 3))]).load_state_dict(_saved(torch.nn.Parameter(rows)))


def test_a_state_dict_may_number_its_parameters_otherwise():
    from medical_image_segmentation_amd.utils.optim import AdamW8
    p, q = _params((5,), (300,))
    opt = AdamW8([p, q])
    a, b = _saved(torch.nn.Parameter(p.detach().clone()), 4), _saved(torch.nn.Parameter(q.detach().clone()), 9)
    groups = opt.state_dict()["param_groups"]
    state = {"state": {7: a["state"][0], 3: b["state"][0]}, "param_groups": [{**groups[0], "params": [7, 3]}]}
    opt.load_state_dict(state)
    assert (opt.state[p]["step"], opt.state[q]["step"]) == (4, 9) and opt.state[q]["exp_avg"].numel() == 384
    state["param_groups"][0]["params"] = [3, 7]
    with pytest.raises(ValueError, match="parameter 3: exp_avg should be 128 bytes"):
        opt.load_state_dict(state)


def test_a_state_without_a_step_replaces_nothing():
    from medical_image_segmentation_amd.utils.optim import AdamW8
    p = _params((300,))[0]
    opt = AdamW8([p], lr=0.5)
    state = _saved(torch.nn.Parameter(p.detach().clone()))
    del state["state"][0]["step"]
    with pytest.raises(ValueError, match="has no step"):
        opt.load_state_dict(state)
    with pytest.raises(ValueError, match="has no exp_avg"):
        opt.load_state_dict({**state, "state": {0: {"step": 3}}})
    assert not opt.state and opt.param_groups[0]["lr"] == 0.5
