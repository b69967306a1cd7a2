"""An optimiser's step whose updates are orthogonalised: for the matrices between the embedding and the head of a model, where `AdamW`
takes the rest.  One call for all of them."""
from __future__ import annotations

import operator
from collections.abc import Sequence

import torch
from torch import Tensor

from .. import ops

__all__ = ["orthogonalize", "muon_step_", "Muon", "muon_param_groups"]

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_ADJUST = {None: 0, "original": 0, "match_rms_adamw": 1}


def _numbers(ns_coefficients, ns_steps, eps) -> tuple[list[float], int, float]:
    if len(ns_coefficients) != 3:
        raise ValueError(f"ns_coefficients are three numbers, got {ns_coefficients}")
    steps = operator.index(ns_steps)
    if not 1 <= steps <= 100:
        raise ValueError(f"ns_steps must be 1 to 100, got {ns_steps}")
    return [float(x) for x in ns_coefficients], steps, float(eps)


def orthogonalize(matrices: Tensor | Sequence[Tensor], *, ns_coefficients: tuple[float, float, float] = NS_COEFFICIENTS, ns_steps: int = 5,
                  eps: float = 1e-7):
    """Newton-Schulz iteration towards the nearest matrices with orthonormal rows (or columns, where there are fewer of them): with
    `X = U / max(|U|, eps)` (Frobenius norm), `ns_steps` times `A = X X^T; X = a X + (b A + c A A) X`.  The singular vectors stay, each singular
    value s moves by `a s + b s^3 + c s^5`; the usual coefficients bring all but the smallest to between 0.7 and 1.2 in five steps.

    `matrices` is one tensor `[..., m, n]` or a list of them (then a list is returned), in fp32, bf16 or fp16, all on one GPU: all in one call.  The
    products hold 22 bits, whatever the type, and sum in fp32: the result is about as near to the exact iteration's as one in plain fp32, before it is rounded
    to its type; its last bits may depend on what else is in the call.  A matrix of zeros gives zeros, one with a NaN or an infinity NaN.  Coefficients with which values of at most 1 would grow
    past 2.5 raise.  Not differentiable."""
    numbers = _numbers(ns_coefficients, ns_steps, eps)
    if isinstance(matrices, Tensor):
        return ops.orthogonalize([matrices], *numbers)[0]
    return ops.orthogonalize(list(matrices), *numbers) if len(matrices) else []


def muon_step_(params: list[Tensor], grads: list[Tensor], momentum_buffers: list[Tensor], *, lr: float | Tensor = 1e-3, weight_decay: float = 0.1,
               momentum: float = 0.95, nesterov: bool = True, ns_coefficients: tuple[float, float, float] = NS_COEFFICIENTS, eps: float = 1e-7,
               ns_steps: int = 5, adjust_lr_fn: str | None = None) -> None:
    """One step on `params` (matrices `[..., m, n]`, contiguous, fp32, bf16 or fp16 with a gradient of their type) in place:

        m = momentum m + (1 - momentum) g,   u = momentum m + (1 - momentum) g   (nesterov; else u = m)
        p = p (1 - lr weight_decay) - lr stretch orthogonalize(u)

    `momentum_buffers` are fp32.  `stretch` is `sqrt(max(1, m / n))` (`adjust_lr_fn` None or "original") or `0.2 sqrt(max(m, n))`
    ("match_rms_adamw", with which learning rates are those of AdamW).  `lr` may be an fp32 number on the GPU.  Parameters are rounded once;
    those in fp32 take their update from products of 22 bits, those in 16 bits from ones of 11: that update is mostly within 2e-3 of the exact one's size, and
    within 1e-2 where its entries are alike but for their sign.  More than five steps, or other coefficients, that would make more of the rounding
    take 22 bits, too.  Matrices of 64 rows (or columns) or fewer go by 64 bits.  Tensors that are written share
    no memory, with each other or with a gradient."""
    if not len(params):
        raise ValueError("muon_step_: no parameters")
    on_gpu = isinstance(lr, Tensor) and lr.is_cuda
    ops.muon_step_(params, grads, momentum_buffers, [], [0.0 if on_gpu else float(lr), float(momentum), float(weight_decay), float(nesterov),
                                                         float(_adjustment(adjust_lr_fn))], [lr] if on_gpu else [],
                   *_numbers(ns_coefficients, ns_steps, eps))


def _adjustment(adjust_lr_fn: str | None) -> int:
    if adjust_lr_fn not in _ADJUST:
        raise ValueError(f"adjust_lr_fn must be None, 'original' or 'match_rms_adamw', got {adjust_lr_fn!r}")
    return _ADJUST[adjust_lr_fn]


def _check_settings(group: dict) -> None:
    if not 0.0 <= float(group["lr"]) or not 0.0 <= group["weight_decay"]:
        raise ValueError(f"lr and weight_decay must not be negative, got {group['lr']}, {group['weight_decay']}")
    if group["adamw"]:
        if not all(0.0 <= b < 1.0 for b in group["betas"]) or not 0.0 <= group["adamw_eps"]:
            raise ValueError(f"betas must be in [0, 1) and adamw_eps not negative, got {group['betas']}, {group['adamw_eps']}")
        return
    if not 0.0 <= group["momentum"] < 1.0:
        raise ValueError(f"momentum must be in [0, 1), got {group['momentum']}")
    if not 1e-30 <= group["eps"] <= 1.0:
        raise ValueError(f"eps must be in [1e-30, 1], got {group['eps']}")
    _numbers(group["ns_coefficients"], group["ns_steps"], group["eps"])
    _adjustment(group["adjust_lr_fn"])
    for p in group["params"]:
        if p.dim() < 2:
            raise ValueError(f"Muon steps matrices, not a parameter of shape {tuple(p.shape)}: put it into a group with adamw=True")


class Muon(torch.optim.Optimizer):
    """Muon whose step is one call for the matrices of all parameter groups (`muon_step_`), for GPU parameters in fp32, bf16 or fp16, with the
    arguments of `torch.optim.Muon`.  Parameters of more than two dimensions are stacks of matrices.

    Groups with `adamw=True` are stepped by `adamw_step_` in the same call of `step`, with `betas` and `adamw_eps`: embeddings, head, norms and
    biases, so that one optimiser (and one learning-rate schedule) serves a whole model; `muon_param_groups` makes such groups, and
    `adjust_lr_fn="match_rms_adamw"` lets both kinds share a learning rate.  A group's `lr` may be an fp32 number on the GPU, and step counters
    live there: a step can be captured into a graph.  Parameters without a gradient are left alone.  Momentum and moments are fp32.  All of a call's
    parameters are on one GPU; it takes up to 8 GiB of workspace, or what the largest matrix needs."""

    def __init__(self, params, lr: float | Tensor = 1e-3, weight_decay: float = 0.1, momentum: float = 0.95, nesterov: bool = True,
                 ns_coefficients: tuple[float, float, float] = NS_COEFFICIENTS, eps: float = 1e-7, ns_steps: int = 5,
                 adjust_lr_fn: str | None = None, *, betas: tuple[float, float] = (0.9, 0.999), adamw_eps: float = 1e-8):
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov, ns_coefficients=ns_coefficients,
                                      eps=eps, ns_steps=ns_steps, adjust_lr_fn=adjust_lr_fn, adamw=False, betas=betas, adamw_eps=adamw_eps))

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        try:
            _check_settings(self.param_groups[-1])
        except ValueError:
            self.param_groups.pop()
            raise

    def _state_of(self, p: Tensor, adamw: bool) -> dict:
        state = self.state[p]
        if not state:
            if adamw:
                state["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
            for k in ("exp_avg", "exp_avg_sq") if adamw else ("momentum_buffer",):
                state[k] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
        return state

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls: dict = {}  # groups of one kind of step, and with the same iteration
        for group in self.param_groups:
            lr = group["lr"]
            on_gpu = isinstance(lr, Tensor) and lr.is_cuda
            number = 0.0 if on_gpu else float(lr)
            if group["adamw"]:
                kind, hyper = None, [number, *map(float, group["betas"]), float(group["adamw_eps"]), float(group["weight_decay"])]
            else:
                kind = (*map(float, group["ns_coefficients"]), operator.index(group["ns_steps"]), float(group["eps"]))
                hyper = [number, float(group["momentum"]), float(group["weight_decay"]), float(group["nesterov"]), float(_adjustment(group["adjust_lr_fn"]))]
            call = calls.setdefault(kind, dict(params=[], grads=[], states=[], of=[], hyper=[], lrs=[]))
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("Muon does not take sparse gradients")
                if not p.is_cuda:
                    raise RuntimeError("Muon steps GPU parameters only")
                call["params"].append(p)
                call["grads"].append(p.grad)
                call["states"].append(self._state_of(p, group["adamw"]))
                call["of"].append(len(call["lrs"]))
            call["hyper"] += hyper
            call["lrs"].append(lr if on_gpu else None)
        for kind, call in calls.items():
            params, states = call["params"], call["states"]
            if not params:
                continue
            none = params[0].new_empty(0, dtype=torch.float32)
            lrs = [none if lr is None else lr for lr in call["lrs"]] if any(lr is not None for lr in call["lrs"]) else []
            if kind is None:
                ops.adamw_step_(params, call["grads"], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                                [s["step"] for s in states], [], [], call["of"], call["hyper"], lrs, -1.0, 0)
            else:
                ops.muon_step_(params, call["grads"], [s["momentum_buffer"] for s in states], call["of"], call["hyper"], lrs,
                               list(kind[:3]), kind[3], kind[4])
        return loss

    def load_state_dict(self, state_dict: dict) -> None:
        """As the base class, hooks included, except that momentum and moments stay (or become) fp32: it would cast them to the parameters'
        types.  The state of a `torch.optim.Muon` is taken too."""
        taken = {}

        def take(_, given):
            self._check_state_dict(given)
            taken.update(given)

        # (behind the caller's hooks of the one kind and before those of the other)
        hooks = [self.register_load_state_dict_pre_hook(take), self.register_load_state_dict_post_hook(lambda _: self._take_state(taken), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _pairs(self, state_dict: dict):
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [(p, g) for g in self.param_groups for p in g["params"]]
        return [(p, g, state_dict["state"].get(i)) for i, (p, g) in zip(ids, params)]

    def _check_state_dict(self, state_dict: dict) -> None:
        for mine, given in zip(self.param_groups, state_dict["param_groups"]):
            if bool(given.get("adamw", False)) != mine["adamw"]:
                raise ValueError("a group of the state is stepped by AdamW and Muon's is not, or the other way round")
        for place, (p, group, saved) in enumerate(self._pairs(state_dict)):
            if not saved:
                continue
            wanted = ("step", "exp_avg", "exp_avg_sq") if group["adamw"] else ("momentum_buffer",)
            missing = [k for k in wanted if k not in saved]
            if missing:
                raise ValueError(f"the state of parameter {place} has {sorted(saved)}, but no {', '.join(missing)}")
            for k in wanted:
                if k != "step" and (saved[k].shape != p.shape or not saved[k].is_floating_point() or saved[k].dtype.itemsize < 2):
                    raise ValueError(f"the {k} of parameter {place} is {saved[k].dtype} {tuple(saved[k].shape)}, the parameter {tuple(p.shape)}")

    def _take_state(self, state_dict: dict) -> None:
        for group in self.param_groups:
            for k, v in self.defaults.items():
                group.setdefault(k, v)
        for p, group, saved in self._pairs(state_dict):
            for k in ("step", "exp_avg", "exp_avg_sq") if group["adamw"] else ("momentum_buffer",):
                if saved and k in saved:
                    t = torch.as_tensor(saved[k]).to(device=p.device, dtype=torch.float32, copy=True)
                    # (in the parameter's order of entries, as the step asks for it, whatever it was saved in)
                    self.state[p][k] = t if k == "step" else torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format).copy_(t)


_HEADS = ("lm_head", "score", "classifier", "qa_outputs")  # as transformers' models call what stands behind their last layer


def _heads(model: torch.nn.Module):
    """The output heads of the model, which may be wrapped (for data-parallel training, or by adapters)."""
    for m in model.modules():
        if m is not model and not hasattr(m, "get_output_embeddings") and not hasattr(m, "get_input_embeddings"):
            continue
        try:
            yield m.get_output_embeddings() if hasattr(m, "get_output_embeddings") else None
        except NotImplementedError:  # (of encoders without one)
            pass
        yield from (getattr(m, name, None) for name in _HEADS)


def muon_param_groups(model: torch.nn.Module) -> list[dict]:
    """Two groups for `Muon`: the model's trainable matrices, and with `adamw=True` its embeddings, its output head (of a language model, or a classifier's)
    and whatever is no matrix (convolutions' weights neither)."""
    kinds = (torch.nn.Embedding, torch.nn.modules.conv._ConvNd)
    apart = {id(p) for m in model.modules() if isinstance(m, kinds) for p in m.parameters(recurse=False)}
    apart |= {id(p) for head in _heads(model) if isinstance(head, torch.nn.Module) for p in head.parameters()}
    params = [p for p in model.parameters() if p.requires_grad]
    matrices = [p for p in params if p.dim() >= 2 and id(p) not in apart]
    chosen = {id(p) for p in matrices}
    return [dict(params=matrices), dict(params=[p for p in params if id(p) not in chosen], adamw=True)]
