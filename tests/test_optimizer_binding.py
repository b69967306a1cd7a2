"""`patch_trl(adamw=True)` on stand-ins for the reference's modules (their trainers are subclasses of `transformers.Trainer`), and the
optimiser's own host logic."""
import sys
import types

import pytest
import torch


@pytest.fixture
def fake_trl(monkeypatch):
    transformers = pytest.importorskip("transformers")
    modules = {name: types.ModuleType(name) for name in ("trl", "trl.trainer", "trl.trainer.utils", "trl.trainer.grpo_trainer",
                                                         "trl.trainer.dpo_trainer")}
    modules["trl.trainer.grpo_trainer"].GRPOTrainer = type("GRPOTrainer", (transformers.Trainer,), {})
    modules["trl.trainer.dpo_trainer"].DPOTrainer = type("DPOTrainer", (transformers.Trainer,), {})
    for name, mod in modules.items():
        if "." in name:
            setattr(modules[name.rsplit(".", 1)[0]], name.rsplit(".", 1)[1], mod)
        mod.__path__ = []
        monkeypatch.setitem(sys.modules, name, mod)
    return modules


def test_patch_binds_the_optimiser(fake_trl, tmp_path):
    import transformers

    import trl_amd
    from trl_amd import integration

    trainers = [fake_trl["trl.trainer.grpo_trainer"].GRPOTrainer, fake_trl["trl.trainer.dpo_trainer"].DPOTrainer]
    make = lambda optim: transformers.TrainingArguments(output_dir=str(tmp_path), optim=optim, learning_rate=3e-4, adam_beta2=0.95,  # noqa: E731
                                                        adam_epsilon=1e-6, use_cpu=True)
    assert integration.patch_trl(grpo=False, adamw=True) == 2
    try:
        for cls in trainers:
            for optim, bits in (("adamw_torch", 32), ("adamw_torch_fused", 32), ("adamw_8bit", 8), ("adamw_bnb_8bit", 8)):
                found, kwargs = cls.get_optimizer_cls_and_kwargs(make(optim))
                assert found is trl_amd.AdamW
                assert kwargs == dict(lr=3e-4, betas=(0.9, 0.95), eps=1e-6, state_bits=bits)
                found([torch.nn.Parameter(torch.zeros(3))], **kwargs)
            assert cls.get_optimizer_cls_and_kwargs(make("sgd"))[0] is torch.optim.SGD
    finally:
        integration.unpatch_trl()
    for cls in trainers:
        assert "get_optimizer_cls_and_kwargs" not in cls.__dict__
        assert cls.get_optimizer_cls_and_kwargs(make("adamw_torch"))[0] is torch.optim.AdamW


def test_optimiser_arguments():
    import trl_amd

    w = torch.nn.Parameter(torch.zeros(3))
    for kw in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(betas=(-0.1, 0.9)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(state_bits=4),
               dict(max_grad_norm=-0.1), dict(max_grad_norm=float("nan"))):
        with pytest.raises(ValueError):
            trl_amd.AdamW([w], **kw)
    opt = trl_amd.AdamW([dict(params=[w], lr=1e-2, weight_decay=0.0)], max_grad_norm=1.0)
    assert opt.param_groups[0]["lr"] == 1e-2 and opt.step() is None and opt.grad_norm is None  # (no gradients: nothing to do)
    schedule = torch.optim.lr_scheduler.LinearLR(opt, 0.1, 1.0, 10)
    assert opt.param_groups[0]["lr"] == pytest.approx(1e-3)
    assert opt.step(lambda: 5.0) == 5.0
    schedule.step()
    assert opt.param_groups[0]["lr"] == pytest.approx(1.9e-3) and opt.state_dict()["state"] == {}


def test_state_of_torch_adamw_is_taken():
    import trl_amd

    theirs = [torch.nn.Parameter(torch.arange(6.0).reshape(2, 3).to(torch.bfloat16)), torch.nn.Parameter(torch.ones(4))]
    opt = torch.optim.AdamW(theirs, lr=1e-2, foreach=False)
    for _ in range(3):
        for w in theirs:
            w.grad = torch.full_like(w, 0.5)
        opt.step()
    saved = opt.state_dict()
    ours = trl_amd.AdamW([torch.nn.Parameter(w.detach().clone()) for w in theirs], lr=1.0, state_bits=8)
    ours.load_state_dict(saved)
    group = ours.param_groups[0]
    assert group["lr"] == 1e-2 and group["state_bits"] == 8 and group["min_8bit_size"] == 4096
    for w, mine in zip(theirs, group["params"]):
        state = ours.state[mine]
        assert set(state) == {"step", "exp_avg", "exp_avg_sq"} and all(v.dtype == torch.float32 for v in state.values())
        assert state["step"].item() == 3.0 and state["step"].shape == ()
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(state[k], opt.state[w][k].float()) and state[k].shape == w.shape
            assert state[k].data_ptr() != opt.state[w][k].data_ptr()
    again = trl_amd.AdamW([torch.nn.Parameter(w.detach().clone()) for w in theirs])
    again.load_state_dict(ours.state_dict())
    assert all(torch.equal(again.state[b][k], ours.state[a][k])
               for a, b in zip(group["params"], again.param_groups[0]["params"]) for k in ("step", "exp_avg", "exp_avg_sq"))
    for kw in (dict(amsgrad=True), dict(maximize=True)):
        with pytest.raises(ValueError, match=next(iter(kw))):
            again.load_state_dict(torch.optim.AdamW(theirs, **kw).state_dict())
