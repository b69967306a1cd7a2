"""The other end of the table that the fused head reads: the embedding of the tokens, times a scale, and its gradient from sorted tokens."""
from __future__ import annotations

import copy
import functools

import torch
from torch import Tensor

from .. import ops

__all__ = ["embedding", "embedding_grad_", "patch_embedding"]


def _padding(padding_idx: int | None, vocab: int) -> int:
    """As `torch.nn.functional.embedding` takes it: negative ones count from the end.  -1: none."""
    if padding_idx is None:
        return -1
    if not -vocab <= padding_idx < vocab:
        raise ValueError(f"padding_idx {padding_idx} is outside a table of {vocab} tokens")
    return padding_idx % vocab


def embedding(input_ids: Tensor, weight: Tensor, *, scale: float = 1.0, padding_idx: int | None = None) -> Tensor:
    """`scale * weight[input_ids]`, rounded once: `[..., H]` in the type of `weight` (`[V, H]`, fp32, bf16 or fp16, rows at any
    stride) for int64 or int32 ids `[...]`.  Differentiable w.r.t. `weight`: the gradient, dense, sums a token's rows in fp32 in
    an order that depends on the ids alone (the same call gives the same bits) and is rounded once; tokens `padding_idx` have none.  A scale that requires
    a gradient raises.

    Ids outside [0, V) give NaN, have no gradient and are reported by `check_device_errors()`."""
    if isinstance(scale, Tensor) and scale.requires_grad and torch.is_grad_enabled():
        raise ValueError("embedding has no gradient for its scale")
    return ops.embedding(input_ids, weight, float(scale), _padding(padding_idx, weight.shape[0]))


def embedding_grad_(grad_weight: Tensor, grad_output: Tensor, input_ids: Tensor, *, scale: float = 1.0,
                    padding_idx: int | None = None) -> Tensor:
    """Adds the gradient that `embedding` has with the upstream gradient `grad_output` (`[..., H]`) to `grad_weight` (`[V, H]`, of that
    type or fp32, rows at any stride) in place, and returns it.  Only the rows of tokens that occur are read and written, each
    entry rounded once: for gradients that are kept by the caller, of a tied head's table or over several micro-batches, where
    a dense gradient would be written, read and added for all V tokens."""
    ops.embedding_grad_(grad_weight, grad_output, input_ids, float(scale), _padding(padding_idx, grad_weight.shape[0]))
    return grad_weight


def _is_lookup_times_scale(module: torch.nn.Embedding) -> bool:
    """Whether the module's forward is its table's rows times `embed_scale` and nothing else: it has no other parameter, and makes just that of every
    token of a narrow table."""
    scale = getattr(module, "embed_scale", None)
    if scale is None or [name for name, _ in module.named_parameters()] != ["weight"]:
        return False
    device = "cpu" if module.weight.is_meta else module.weight.device
    table = (torch.arange(module.num_embeddings, dtype=torch.float32, device=device)[:, None] % 1021 + 1.0) / 512
    probe = copy.copy(module)
    vars(probe)["_parameters"] = {"weight": torch.nn.Parameter(table, requires_grad=False)}
    factor = float(scale.to(table.dtype)) if isinstance(scale, Tensor) else scale
    try:
        with torch.no_grad():
            rows = type(module).forward(probe, torch.arange(module.num_embeddings, device=device)[None])
    except Exception:
        return False
    return isinstance(rows, Tensor) and torch.equal(rows, (table * factor)[None])


def _is_scaled(module: torch.nn.Embedding) -> bool:
    """Whether the module's forward multiplies its rows by `embed_scale`.  ValueError where it is neither that nor a lookup."""
    if type(module).forward is torch.nn.Embedding.forward:
        return False
    if not type(module).__name__.endswith("ScaledWordEmbedding") or not _is_lookup_times_scale(module):
        raise ValueError(f"{type(module).__name__} is not a lookup, or a scaled one, that patch_embedding knows")
    return True


def _scale_of(module: torch.nn.Embedding) -> float:
    """The factor that the module multiplies its rows by now.  As a tensor it is rounded to the table's type before it is multiplied with, and casts of the
    model change both; its number is read again, which waits for the GPU, where the tensor is another one or has changed."""
    scale = module.embed_scale
    if not isinstance(scale, Tensor):
        return float(scale)
    seen = 0 if scale.is_inference() else scale._version, module.weight.dtype
    held = vars(module).get("_trl_amd_scale")
    if held is None or held[0] is not scale or held[1] != seen:
        held = vars(module)["_trl_amd_scale"] = scale, seen, float(scale.detach().to(module.weight.dtype))
    return held[2]


def _embedding_forward(module: torch.nn.Embedding, input: Tensor) -> Tensor:
    if not module._trl_amd_scaled:
        return embedding(input, module.weight, padding_idx=module.padding_idx)
    if torch.compiler.is_compiling() and isinstance(module.embed_scale, Tensor):  # (its number is not to be had while a graph is made)
        return embedding(input, module.weight, padding_idx=module.padding_idx) * module.embed_scale.to(module.weight.dtype)
    return embedding(input, module.weight, scale=_scale_of(module), padding_idx=module.padding_idx)


def patch_embedding(model: torch.nn.Module) -> None:
    """Replaces the forward of `model.get_input_embeddings()` by `embedding`, with the module's own scale (as it is at each call) and padding index.  Takes
    `torch.nn.Embedding` and the scaled embeddings of transformers' models whose forward is the rows times `embed_scale` and nothing else (it
    is run once, on a narrow table); others, embeddings with `max_norm`, `sparse` or `scale_grad_by_freq`, and modules whose forward
    has been replaced already, raise ValueError."""
    module = model.get_input_embeddings()
    if not isinstance(module, torch.nn.Embedding):
        raise ValueError(f"the model's input embeddings are a {type(module).__name__}, not a torch.nn.Embedding")
    if module.max_norm is not None or module.sparse or module.scale_grad_by_freq:
        raise ValueError("patch_embedding takes no max_norm, sparse or scale_grad_by_freq")
    own = vars(module).get("forward")
    if own is not None and getattr(own, "func", None) is not _embedding_forward:
        raise ValueError("the input embeddings' forward has been replaced already, by a hook for instance: patch_embedding would drop it, call it first")
    module._trl_amd_scaled = _is_scaled(module)
    if module._trl_amd_scaled:
        _scale_of(module)  # (read now, not in the first forward)
    # (a copy of the model gets one of its own table, and one that has been pickled, too, which a bound method does not survive)
    module.forward = functools.partial(_embedding_forward, module)
