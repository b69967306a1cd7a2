"""Which models `patch_trl(adamw=True)` gives `trl_amd.AdamW` to: those whose parameters one call of it can step.  Others keep the optimiser
that they would have had."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from test_optimizer_binding import fake_trl  # noqa: F401  (the fixture)


def model(device, dtype=torch.float32, head=None):
    return torch.nn.Sequential(torch.nn.Embedding(100, 64, device=device, dtype=dtype), torch.nn.Linear(64, 100, device=head or device, dtype=dtype))


@pytest.fixture
def patched(fake_trl, tmp_path):  # noqa: F811
    import transformers

    from trl_amd import integration

    assert integration.patch_trl(grpo=False, adamw=True) == 2
    args = lambda optim="adamw_torch": transformers.TrainingArguments(output_dir=str(tmp_path), optim=optim, use_cpu=True, report_to=[])  # noqa: E731
    yield fake_trl["trl.trainer.grpo_trainer"].GRPOTrainer, args
    integration.unpatch_trl()


def test_a_trainer_on_the_cpu_steps(patched):
    cls, args = patched
    trainer = cls(model=model("cpu"), args=args())
    opt = trainer.create_optimizer()
    assert type(opt) is torch.optim.AdamW
    for p in trainer.model.parameters():
        p.grad = torch.ones_like(p)
    opt.step()


def test_models_that_one_call_steps_and_others(patched):
    import trl_amd

    cls, args = patched
    with FakeTensorMode():
        one, two, double = model("cuda:0"), model("cuda:0", head="cuda:1"), model("cuda:0", torch.float64)
        frozen = model("cpu", torch.bfloat16, head="cuda:0")
        frozen[0].requires_grad_(False)
    found = lambda m: cls.get_optimizer_cls_and_kwargs(args(), m)[0]  # noqa: E731
    assert found(one) is trl_amd.AdamW and found(frozen) is trl_amd.AdamW
    for m in (two, double, model("cpu"), model("meta")):
        assert found(m) is torch.optim.AdamW
    assert found(None) is trl_amd.AdamW  # (nothing is known)


def test_sharded_parameters_keep_their_optimiser(patched):
    from torch.testing._internal.two_tensor import TwoTensor  # a wrapper of other tensors, as sharded parameters are

    cls, args = patched
    with FakeTensorMode():
        sharded = model("cuda:0")
        w = sharded[1].weight.detach()
        sharded[1].weight = torch.nn.Parameter(TwoTensor(w, w.clone()))
    assert cls.get_optimizer_cls_and_kwargs(args(), sharded)[0] is torch.optim.AdamW


def test_embeddings_keep_fp32_moments(patched):
    """The 8-bit optimisers behind these names hold embeddings' moments in 32 bits."""
    import copy

    import trl_amd

    cls, args = patched
    with FakeTensorMode():
        m = model("cuda:0")
        m[1].weight = torch.nn.Parameter(torch.empty(100, 64, device="cuda:0"))
        for optim in ("adamw_8bit", "adamw_bnb_8bit"):
            found, kwargs = cls.get_optimizer_cls_and_kwargs(args(optim), m)
            assert found is trl_amd.AdamW and kwargs["state_bits"] == 8
            opt = found(m.parameters(), **kwargs)
            kinds = {n: opt._state_of(p, opt.param_groups[0])["exp_avg"].dtype for n, p in m.named_parameters()}
            assert kinds == {"0.weight": torch.float32, "1.weight": torch.float8_e4m3fn, "1.bias": torch.float32}
        assert "keep_32bit" not in cls.get_optimizer_cls_and_kwargs(args(), m)[1]
    w = [torch.nn.Parameter(torch.zeros(5000)) for _ in range(2)]
    opt = copy.deepcopy(trl_amd.AdamW(w, state_bits=8, keep_32bit=w[:1]))
    kinds = [opt._state_of(p, opt.param_groups[0])["exp_avg"].dtype for p in opt.param_groups[0]["params"]]
    assert kinds == [torch.float32, torch.float8_e4m3fn]
