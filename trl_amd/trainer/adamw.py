"""The optimiser's step of the reference's training loop (`transformers.Trainer` with `optim="adamw_torch"` or an 8-bit AdamW, and
`max_grad_norm`): one call for all tensors of a model."""
from __future__ import annotations

from collections.abc import Iterable

import torch
from torch import Tensor
from torch.utils._python_dispatch import is_traceable_wrapper_subclass

from .. import ops

__all__ = ["adamw_step_", "adamw_state_values", "AdamW", "optimizer_cls_and_kwargs"]

STATE_BLOCK = 256  # entries of 8-bit moments that share a scale


def adamw_step_(params: list[Tensor], grads: list[Tensor], exp_avgs: list[Tensor], exp_avg_sqs: list[Tensor], steps: list[Tensor], *,
                lr: float | Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                max_grad_norm: float | None = None, exp_avg_scales: list[Tensor] | None = None,
                exp_avg_sq_scales: list[Tensor] | None = None, seed: int = 0) -> Tensor | None:
    """One AdamW step on `params` in place, each in fp32, bf16 or fp16 with a gradient of its type.  The arithmetic is
    `torch.optim.AdamW`'s, in fp32; parameters are rounded once to their type.  `steps` (fp32, one number each, on the GPU) count
    up first.  `lr` may be an fp32 number on the GPU.  Tensors that are written share no memory, with each other or with a gradient.

    With `max_grad_norm` the gradients count as multiplied by `min(1, max_grad_norm / (norm + 1e-6))`, `norm` the 2-norm of all of
    them, as `torch.nn.utils.clip_grad_norm_` does (which writes them; they stay as they are here), and the norm is returned (fp32,
    on the GPU).  0 returns the norm and clips nothing.

    `exp_avgs` and `exp_avg_sqs` are fp32, or float8_e4m3fn and uint8 codes with fp32 scales, one for each 256 entries (`AdamW`
    makes them; all zeros is a valid start).  Codes round up or down by bits that are a hash of `seed`, the step, the parameter's
    place in the list and the entry: the same call gives the same state."""
    on_gpu = isinstance(lr, Tensor) and lr.is_cuda
    norm = ops.adamw_step_(params, grads, exp_avgs, exp_avg_sqs, steps, exp_avg_scales or [], exp_avg_sq_scales or [], [],
                           [0.0 if on_gpu else float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay)],
                           [lr] if on_gpu else [], -1.0 if max_grad_norm is None else _clip(max_grad_norm), seed & 0xFFFFFFFF)
    return None if max_grad_norm is None else norm


def _clip(max_grad_norm: float) -> float:
    if not max_grad_norm >= 0:
        raise ValueError(f"max_grad_norm must not be negative, got {max_grad_norm}")
    return float(max_grad_norm)


def adamw_state_values(codes: Tensor, scales: Tensor) -> Tensor:
    """The values of 8-bit moments, exact in bf16, in the shape of `codes`."""
    return ops.adamw_state_values(codes, scales)


def _check_settings(lr, betas, eps, weight_decay, state_bits) -> None:
    if state_bits not in (8, 32):
        raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
    if not 0.0 <= float(lr) or not 0.0 <= eps or not 0.0 <= weight_decay:
        raise ValueError(f"lr, eps and weight_decay must not be negative, got {lr}, {eps}, {weight_decay}")
    if not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0:
        raise ValueError(f"betas must be in [0, 1), got {betas}")


class AdamW(torch.optim.Optimizer):
    """AdamW whose step is one call for all parameter groups (`adamw_step_`), for GPU parameters in fp32, bf16 or fp16.

    `state_bits=8` holds both moments of every parameter of `min_8bit_size` entries or more in 8 bits, 2.03 bytes per entry instead
    of 8, but for those in `keep_32bit`.  With `max_grad_norm` the step clips the norm over all groups (of this process's tensors), without a
    pass that writes the gradients, and leaves it in `grad_norm` (fp32, on the GPU); `transformers.Trainer` then runs with `max_grad_norm=0`.
    Step counters live on the GPU and a group's `lr` may: a step can be captured into a graph.  Parameters without a gradient are left alone; the
    others lie on one GPU.  Moments are fp32 (or in 8 bits) whatever the parameters' type."""

    def __init__(self, params, lr: float | Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, *, state_bits: int = 32, min_8bit_size: int = 4096, max_grad_norm: float | None = None,
                 seed: int = 0, keep_32bit: Iterable[Tensor] = ()):
        _check_settings(lr, betas, eps, weight_decay, state_bits)
        self.max_grad_norm = None if max_grad_norm is None else _clip(max_grad_norm)
        self.seed, self.grad_norm, self.keep_32bit = int(seed), None, set(keep_32bit)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      min_8bit_size=min_8bit_size))

    def add_param_group(self, param_group: dict) -> None:
        _check_settings(**{k: param_group.get(k, self.defaults[k]) for k in ("lr", "betas", "eps", "weight_decay", "state_bits")})
        super().add_param_group(param_group)

    def __getstate__(self) -> dict:
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm, "seed": self.seed, "grad_norm": self.grad_norm,
                "keep_32bit": self.keep_32bit}

    def _state_of(self, p: Tensor, group: dict) -> dict:
        state = self.state[p]
        if not state:
            state["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
            if group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"] and p not in self.keep_32bit:
                blocks = -(-p.numel() // STATE_BLOCK)
                state["exp_avg"] = torch.zeros_like(p, dtype=torch.uint8, memory_format=torch.preserve_format).view(torch.float8_e4m3fn)
                state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.uint8, memory_format=torch.preserve_format)
                state["exp_avg_scale"] = torch.ones(blocks, dtype=torch.float32, device=p.device)
                state["exp_avg_sq_scale"] = torch.ones(blocks, dtype=torch.float32, device=p.device)
            else:
                state["exp_avg"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
                state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
        return state

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        params, grads, states, group_of, hyper, lrs = [], [], [], [], [], []
        for i, group in enumerate(self.param_groups):
            lr = group["lr"]
            on_gpu = isinstance(lr, Tensor) and lr.is_cuda
            hyper += [0.0 if on_gpu else float(lr), *map(float, group["betas"]), float(group["eps"]), float(group["weight_decay"])]
            lrs.append(lr if on_gpu else None)
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not take sparse gradients")
                if not p.is_cuda:
                    raise RuntimeError("AdamW steps GPU parameters only")
                params.append(p)
                grads.append(p.grad)
                states.append(self._state_of(p, group))
                group_of.append(i)
        self.grad_norm = None
        if not params:
            return loss
        none = params[0].new_empty(0, dtype=torch.float32)
        scales = [[s.get(k, none) for s in states] for k in ("exp_avg_scale", "exp_avg_sq_scale")]
        norm = ops.adamw_step_(params, grads, [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                               [s["step"] for s in states], *scales, group_of, hyper,
                               [none if lr is None else lr for lr in lrs] if any(lr is not None for lr in lrs) else [],
                               -1.0 if self.max_grad_norm is None else self.max_grad_norm, self.seed & 0xFFFFFFFF)
        self.grad_norm = None if self.max_grad_norm is None else norm
        return loss

    def load_state_dict(self, state_dict: dict) -> None:
        """As the base class, hooks included, except that the moments keep their own types (it would cast them to the parameters').  The
        state of a `torch.optim.AdamW` is taken too: its moments become fp32 and its step counters move to the parameters' device."""
        taken = {}

        def take(_, given):
            self._check_state_dict(given)
            taken.update(given)

        # (behind the caller's hooks of the one kind and before those of the other: what a pre-hook returns is what is loaded, and a post-hook
        # finds the state as it will be)
        hooks = [self.register_load_state_dict_pre_hook(take),
                 self.register_load_state_dict_post_hook(lambda _: self._take_state(taken), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _check_state_dict(self, state_dict: dict) -> None:
        """Refuses what would not go on as it was: another optimiser's state, or another kind of step."""
        for group in state_dict["param_groups"]:
            for k in ("amsgrad", "maximize"):
                if group.get(k):
                    raise ValueError(f"AdamW has no {k}")
            if group.get("decoupled_weight_decay") is False and group.get("weight_decay"):
                raise ValueError("AdamW's weight decay is decoupled, the state's is not")
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for place, (i, p) in enumerate(zip(ids, params)):
            saved = state_dict["state"].get(i)
            if not saved:
                continue
            missing = [k for k in ("step", "exp_avg", "exp_avg_sq") if k not in saved]
            if missing:
                raise ValueError(f"the state of parameter {place} is not AdamW's: it has {sorted(saved)}, but no {', '.join(missing)}")
            scales = [saved[k] for k in ("exp_avg_scale", "exp_avg_sq_scale") if k in saved]
            kinds = saved["exp_avg"].dtype, saved["exp_avg_sq"].dtype
            coded = kinds == (torch.float8_e4m3fn, torch.uint8)
            if len(scales) != 2 * coded or not coded and any(k.itemsize == 1 for k in kinds):
                raise ValueError(f"the state of parameter {place} has moments in {kinds[0]} and {kinds[1]} and {len(scales)} scales")
            if any(saved[k].shape != p.shape for k in ("exp_avg", "exp_avg_sq")) or any(t.numel() != -(-p.numel() // STATE_BLOCK) for t in scales):
                raise ValueError(f"the state of parameter {place} is that of another shape than {tuple(p.shape)}")

    def _take_state(self, state_dict: dict) -> None:
        """The moments and step counters of `state_dict`, which the base class has loaded, in their own types."""
        for group in self.param_groups:
            for k, v in self.defaults.items():
                group.setdefault(k, v)
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            saved = state_dict["state"].get(i, {})
            for k in ("step", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
                if k in saved:
                    t = torch.as_tensor(saved[k]).to(device=p.device, copy=True)
                    self.state[p][k] = t if "exp_avg_scale" in saved else t.float()


_STATE_BITS = {"adamw_torch": 32, "adamw_torch_fused": 32, "adamw_8bit": 8, "adamw_bnb_8bit": 8}  # names of `TrainingArguments.optim`


def _steps_all_of(model: torch.nn.Module) -> bool:
    """Whether one call can step the model's trainable parameters: plain tensors of its types on one GPU (sharded ones are none)."""
    params = [p for p in model.parameters() if p.requires_grad]
    return (len({p.device for p in params}) == 1 and params[0].is_cuda and not any(map(is_traceable_wrapper_subclass, params))
            and all(p.dtype in (torch.float32, torch.bfloat16, torch.float16) for p in params))


def optimizer_cls_and_kwargs(args, model: torch.nn.Module | None = None) -> tuple[type, dict] | None:
    """`AdamW` and its arguments for training arguments whose `optim` is an AdamW, plain or with 8-bit states; `None` for others, and for
    a model that it cannot step (on the CPU, on several GPUs, with sharded parameters or in another type).  What
    `transformers.Trainer.get_optimizer_cls_and_kwargs` returns, and its trainers take as `optimizer_cls_and_kwargs`."""
    bits = _STATE_BITS.get(getattr(args.optim, "value", args.optim))
    if bits is None or model is not None and not _steps_all_of(model):
        return None
    kwargs = dict(lr=args.learning_rate, betas=(args.adam_beta1, args.adam_beta2), eps=args.adam_epsilon, state_bits=bits)
    if bits == 8 and model is not None:  # (as the trainers have it of the optimiser that they know by these names)
        kwargs["keep_32bit"] = [m.weight for m in model.modules() if isinstance(m, torch.nn.Embedding)]
    return AdamW, kwargs
