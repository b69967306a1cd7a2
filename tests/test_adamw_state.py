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
