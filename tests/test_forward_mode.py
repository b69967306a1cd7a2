"""Forward mode: the operators have no tangent formula, so a call on dual tensors (or under `torch.func.jvp`) raises, also where nothing
requires a gradient; none returns as if the derivative were zero.  On fake tensors: shapes are enough."""
import pytest
import torch
import torch.autograd.forward_ad as fad
from torch._subclasses.fake_tensor import FakeTensorMode

B, T, V = 4, 5, 64


def calls(dtype):
    import trl_amd

    ids = torch.zeros(B, T, dtype=torch.long, device="cuda")
    mask = torch.ones(B, T, device="cuda")
    row = torch.zeros(B, device="cuda")
    logits = torch.empty(B, T, V, dtype=dtype, device="cuda")
    logp = torch.empty(B, T, device="cuda")
    if dtype == torch.float64:
        return {"selective_log_softmax": (lambda x: trl_amd.selective_log_softmax(x, ids), logits)}
    return {
        "filtered_logps": (lambda x: trl_amd.filtered_logps(x, ids, 0.7, 5, 0.9), logits),
        "selective_log_softmax": (lambda x: trl_amd.selective_log_softmax(x, ids), logits),
        "logps_and_entropies": (lambda x: trl_amd.logps_and_entropies(x, ids)[0], logits),
        "entropy_from_logits": (lambda x: trl_amd.entropy_from_logits(x), logits),
        "grpo_loss": (lambda x: trl_amd.grpo_loss(x, row, mask, num_items_in_batch=20.0)[0], logp),
        "grpo_loss_advantages": (lambda x: trl_amd.grpo_loss(logp, x, mask, num_items_in_batch=20.0)[0], row),
        "rloo_loss": (lambda x: trl_amd.rloo_loss(x, mask, row, row, 0.2, 0.2)[0], logp),
        "dpo_sigmoid_loss": (lambda x: trl_amd.dpo_sigmoid_loss(x, mask, row[: B // 2], row[: B // 2], 0.1)[0], logp),
    }


CASES = [("bf16", n) for n in ("filtered_logps", "selective_log_softmax", "logps_and_entropies", "entropy_from_logits", "grpo_loss",
                               "grpo_loss_advantages", "rloo_loss", "dpo_sigmoid_loss")] + [("fp64", "selective_log_softmax")]


@pytest.mark.parametrize("dtype,name", CASES)
@pytest.mark.parametrize("how", ["plain", "requires_grad", "no_grad", "jvp"])
def test_forward_mode_raises(dtype, name, how):
    with FakeTensorMode():
        call, x = calls({"bf16": torch.bfloat16, "fp64": torch.float64}[dtype])[name]
        call(x)  # (without a tangent it works)
        with pytest.raises((RuntimeError, NotImplementedError)):
            if how == "jvp":
                torch.func.jvp(call, (x,), (torch.empty_like(x),))
            else:
                with fad.dual_level():
                    dual = fad.make_dual(x.requires_grad_(how != "plain"), torch.empty_like(x))
                    if how == "no_grad":
                        with torch.no_grad():
                            call(dual)
                    else:
                        call(dual)


@pytest.mark.parametrize("name", ["filtered_logps", "selective_log_softmax", "rloo_loss", "dpo_sigmoid_loss"])
def test_operands_without_a_tangent_are_taken_at_a_dual_level(name):
    with FakeTensorMode(), fad.dual_level():
        call, x = calls(torch.bfloat16)[name]
        assert call(x).shape == call(x.requires_grad_()).shape and call(x).requires_grad


def test_settings_have_no_derivative():
    """A setting with a value for each row that wants a gradient, or has a tangent, is refused: it would get none, without an error."""
    import trl_amd

    with FakeTensorMode():
        logits, ids = torch.empty(B, V, device="cuda", requires_grad=True), torch.zeros(B, dtype=torch.long, device="cuda")
        for name in ("temperature", "top_p", "min_p"):
            t = torch.full((B,), 0.5, device="cuda")
            assert trl_amd.filtered_logps(logits, ids, **{name: t}).requires_grad
            with fad.dual_level(), pytest.raises(RuntimeError, match="detach"):
                trl_amd.filtered_logps(logits.detach(), ids, **{name: fad.make_dual(t, t)})
            t.requires_grad_()
            for x in (logits, logits.detach()):
                with pytest.raises(RuntimeError, match="detach"):
                    trl_amd.filtered_logps(x, ids, **{name: t})
            assert trl_amd.filtered_logps(logits, ids, **{name: t.detach()}).requires_grad
            with torch.no_grad():
                trl_amd.filtered_logps(logits, ids, **{name: t})
