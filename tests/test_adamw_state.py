"""The state of `AdamW`: loading, hooks around it.  Host logic only."""
import pytest
import torch


def optimiser(state_bits=32, **kw):
    import trl_amd

    w = [torch.nn.Parameter(torch.arange(6.0).reshape(2, 3).to(torch.bfloat16)), torch.nn.Parameter(torch.ones(5000))]
    return w, trl_amd.AdamW(w, lr=1e-2, state_bits=state_bits, **kw)


def torch_state():
    w = [torch.nn.Parameter(torch.arange(6.0).reshape(2, 3).to(torch.bfloat16)), torch.nn.Parameter(torch.ones(5000))]
    opt = torch.optim.AdamW(w, lr=1e-2, foreach=False)
    for _ in range(2):
        for p in w:
            p.grad = torch.full_like(p, 0.5)
        opt.step()
    return opt.state_dict()


def test_what_a_pre_hook_returns_is_loaded():
    w, opt = optimiser()

    def twice(_, state_dict):
        state = {i: {**s, "exp_avg": 2 * s["exp_avg"]} for i, s in state_dict["state"].items()}
        return {**state_dict, "state": state}

    saved = torch_state()
    opt.register_load_state_dict_pre_hook(twice)
    opt.load_state_dict(saved)
    for i, p in enumerate(w):
        assert torch.equal(opt.state[p]["exp_avg"], 2 * saved["state"][i]["exp_avg"].float())
        assert torch.equal(opt.state[p]["exp_avg_sq"], saved["state"][i]["exp_avg_sq"].float())


def test_what_a_post_hook_writes_stays():
    w, opt = optimiser()
    seen = []

    def zero(optimizer):
        for p in w:
            seen.append(optimizer.state[p]["exp_avg"].dtype)
            optimizer.state[p]["exp_avg_sq"] = torch.zeros_like(optimizer.state[p]["exp_avg_sq"])
            optimizer.state[p]["mine"] = 1

    opt.register_load_state_dict_post_hook(zero)
    opt.load_state_dict(torch_state())
    assert seen == [torch.float32] * 2  # (a hook sees the moments in their own types)
    for p in w:
        assert not opt.state[p]["exp_avg_sq"].any() and opt.state[p]["mine"] == 1 and opt.state[p]["exp_avg"].any()
    opt.load_state_dict(torch_state())  # (again: no hook of the first call is left)
    assert seen == [torch.float32] * 4 and len(opt._optimizer_load_state_dict_pre_hooks) == 0 and len(opt._optimizer_load_state_dict_post_hooks) == 1


def bad_states():
    good = torch_state()
    one = lambda entry: {**good, "state": {**good["state"], 1: entry}}  # noqa: E731
    moments = good["state"][1]
    codes = {"step": torch.tensor(1.0), "exp_avg": torch.zeros(5000, dtype=torch.uint8).view(torch.float8_e4m3fn),
             "exp_avg_sq": torch.zeros(5000, dtype=torch.uint8)}
    return {
        "another optimiser's moments": one({"step": 7, "state1": torch.zeros(5000), "state2": torch.zeros(5000)}),
        "momentum": one({"momentum_buffer": torch.zeros(5000)}),
        "no step": one({k: v for k, v in moments.items() if k != "step"}),
        "no second moment": one({k: v for k, v in moments.items() if k != "exp_avg_sq"}),
        "one scale": one({**codes, "exp_avg_scale": torch.ones(20)}),
        "codes without scales": one(codes),
        "scales of fp32 moments": one({**moments, "exp_avg_scale": torch.ones(20), "exp_avg_sq_scale": torch.ones(20)}),
        "another shape": one({**moments, "exp_avg": torch.zeros(4999)}),
        "scales of another size": one({**codes, "exp_avg_scale": torch.ones(19), "exp_avg_sq_scale": torch.ones(20)}),
    }


@pytest.mark.parametrize("what", list(bad_states()))
def test_states_that_are_none_of_its_own_are_refused(what):
    w, opt = optimiser()
    opt.load_state_dict(torch_state())
    before = {p: {k: v.clone() for k, v in opt.state[p].items()} for p in w}
    with pytest.raises(ValueError, match="parameter 1"):
        opt.load_state_dict(bad_states()[what])
    for p in w:  # (and what was there stays)
        assert set(opt.state[p]) == set(before[p]) and all(torch.equal(opt.state[p][k], v) for k, v in before[p].items())


def test_coupled_decay_is_refused():
    w, opt = optimiser()
    saved = torch_state()
    saved["param_groups"][0]["decoupled_weight_decay"] = False
    with pytest.raises(ValueError, match="decoupled"):
        opt.load_state_dict(saved)
    saved["param_groups"][0]["weight_decay"] = 0.0  # (no decay: the two are the same)
    opt.load_state_dict(saved)
    assert opt.state[w[1]]["step"].item() == 2.0


def test_a_hook_may_convert_a_state():
    """What is refused is what the hooks leave."""
    w, opt = optimiser()
    saved = bad_states()["another optimiser's moments"]

    def convert(_, given):
        names = {"state1": "exp_avg", "state2": "exp_avg_sq"}
        return {**given, "state": {i: {names.get(k, k): v for k, v in s.items()} for i, s in given["state"].items()}}

    opt.register_load_state_dict_pre_hook(convert)
    opt.load_state_dict(saved)
    assert opt.state[w[1]]["step"].item() == 7.0 and opt.state[w[1]]["exp_avg"].shape == (5000,)


def test_8bit_state_round_trip_and_empty_entries():
    w, opt = optimiser(8)
    for p in w:
        opt._state_of(p, opt.param_groups[0])
    opt.state[w[1]]["exp_avg_sq"].fill_(7)
    other, again = optimiser(8)
    again.load_state_dict(opt.state_dict())
    assert again.state[other[1]]["exp_avg"].dtype == torch.float8_e4m3fn and bool((again.state[other[1]]["exp_avg_sq"] == 7).all())
    saved = opt.state_dict()
    saved["state"][0] = {}  # (a parameter that has made no step)
    again.load_state_dict(saved)
    assert not again.state[other[0]] and again.state[other[1]]["exp_avg"].dtype == torch.float8_e4m3fn


def test_copies_and_pickles_are_whole():
    import copy
    import pickle

    w, opt = optimiser(max_grad_norm=0.5, seed=9)
    opt.load_state_dict(torch_state())
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert (other.max_grad_norm, other.seed, other.grad_norm) == (0.5, 9, None)
        (a, b) = other.param_groups[0]["params"]
        assert torch.equal(a, w[0]) and torch.equal(other.state[b]["exp_avg"], opt.state[w[1]]["exp_avg"])
        assert other.step() is None  # (no gradients: nothing to do)


def test_what_looks_on_sees_the_operator(monkeypatch):
    """The way past the dispatcher is for calls that nobody watches: under a function mode or a profiler the operator itself is called."""
    import torch.overrides

    from trl_amd import _lib, ops

    taken = []
    monkeypatch.setattr(_lib, "py_adamw_step", lambda args: taken.append("entry point") or torch.zeros(()))
    monkeypatch.setattr(ops, "_adamw_step_op", lambda *args: taken.append("operator") or torch.zeros(()))

    class Mode(torch.overrides.TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    ops.adamw_step_()
    with Mode():
        ops.adamw_step_()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]):
        ops.adamw_step_()
    ops.adamw_step_()
    assert taken == ["entry point", "operator", "operator", "entry point"]
    monkeypatch.delattr(torch._C, "_len_torch_function_stack")  # (a torch that does not answer)
    ops.adamw_step_()
    assert taken[4:] == ["operator"]


def test_operands_that_share_memory_are_refused():
    """Two workgroups would write the same entries.  (On the host: the check comes before that of the device.)"""
    import trl_amd

    def call(p=None, g=None, m=None, v=None, s=None, **kw):
        new = lambda: [torch.zeros(600) for _ in range(2)]  # noqa: E731
        trl_amd.adamw_step_(p or new(), g or new(), m or new(), v or new(), s or [torch.zeros(()) for _ in range(2)], **kw)

    x, y = torch.zeros(600), torch.zeros(600)
    flat = torch.zeros(1801)
    apart, over = [flat[:600], flat[600:1200]], [flat[:600], flat[599:1199]]
    for ok in (dict(), dict(p=apart), dict(m=apart), dict(p=[flat[1201:], flat[:600]], v=[flat[600:1200], y]), dict(g=[x, x]), dict(g=over),
               dict(g=[flat[:600], x], p=[flat[600:1200], y])):
        with pytest.raises(RuntimeError, match="not on a GPU"):
            call(**ok)
    step = torch.zeros(())
    for bad in (dict(p=[x, x]), dict(p=over), dict(m=[x, x]), dict(v=over), dict(s=[step, step]), dict(m=[x, y], v=[y, x]), dict(p=[x, y], m=[y, flat[:600]]),
                dict(p=[x, y], g=[y, x]), dict(p=apart, g=[flat[300:900], x]), dict(p=[flat[1:601], y], s=[flat[0], flat[600]])):
        with pytest.raises(ValueError, match="twice|share"):
            call(**bad)
    codes = [torch.zeros(600, dtype=torch.uint8) for _ in range(4)]
    eight = dict(m=[c.view(torch.float8_e4m3fn) for c in codes[:2]], v=codes[2:])
    scales = [torch.ones(3) for _ in range(4)]
    with pytest.raises(RuntimeError, match="not on a GPU"):
        call(**eight, exp_avg_scales=scales[:2], exp_avg_sq_scales=scales[2:])
    with pytest.raises(ValueError, match="twice|share"):
        call(**eight, exp_avg_scales=scales[:2], exp_avg_sq_scales=[scales[2], scales[0]])
    with pytest.raises(ValueError, match="twice|share"):
        call(m=eight["m"], v=[codes[0], codes[2]], exp_avg_scales=scales[:2], exp_avg_sq_scales=scales[2:])
    none = torch.zeros(0)
    with pytest.raises(RuntimeError, match="not on a GPU"):  # (an empty tensor shares nothing, and stands for no scale)
        call([none, none], [none, none], [none, none], [none, none], exp_avg_scales=[none, none], exp_avg_sq_scales=[none, none])
    one = torch.ones(1)
    with pytest.raises(RuntimeError, match="not on a GPU"):  # (scales of fp32 moments are not looked at)
        call(exp_avg_scales=[one, one], exp_avg_sq_scales=[one, one])


def test_groups_of_their_own_settings():
    import trl_amd

    w = [torch.nn.Parameter(torch.zeros(5000)) for _ in range(2)]
    opt = trl_amd.AdamW([dict(params=w[:1], state_bits=8), dict(params=w[1:])])
    kinds = [opt._state_of(p, g)["exp_avg"].dtype for g in opt.param_groups for p in g["params"]]
    assert kinds == [torch.float8_e4m3fn, torch.float32]
    for bad in (dict(state_bits=16), dict(state_bits="8"), dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-1.0), dict(betas=(0.9, 1.0))):
        with pytest.raises(ValueError):
            trl_amd.AdamW([dict(params=w, **bad)])
        with pytest.raises(ValueError):
            trl_amd.AdamW(w[:1]).add_param_group(dict(params=w[1:], **bad))


def test_other_entries_of_a_state_are_loaded_as_by_the_base_class():
    w, opt = optimiser()
    saved = torch_state()
    saved["state"][1]["seen"] = 17
    saved["state"][0]["step"] = 2  # (a number instead of a tensor)
    opt.load_state_dict(saved)
    assert opt.state[w[1]]["seen"] == 17 and opt.state_dict()["state"][1]["seen"] == 17
    assert opt.state[w[0]]["step"].dtype == torch.float32 and opt.state[w[0]]["step"].item() == 2.0
