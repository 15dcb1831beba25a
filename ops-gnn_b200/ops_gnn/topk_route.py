"""Routing of rows to their best experts.  An addition: the reference has no counterpart; its operators start from edges
that are already there, this one makes them from scores."""
from typing import Optional, Tuple

import torch

from . import _pybind

_SUPPORTED_DTYPES = (torch.float16, torch.float32, torch.bfloat16)
_SCORES = {"softmax": 0, "sigmoid": 1}
MAX_EXPERTS, MAX_CHOSEN, MAX_GROUPS = 1024, 32, 32


def _check_int(name: str, value, low: int, high: int) -> None:
    if type(value) is int and low <= value <= high:
        return
    if not isinstance(value, int) or isinstance(value, bool):
        raise TypeError(f"{name} must be an int, got {type(value).__name__}")
    if not low <= value <= high:
        raise ValueError(f"{name} must be in [{low}, {high}], got {value}")


def topk_route(logits: torch.Tensor, k: int, score: str = "softmax", bias: Optional[torch.Tensor] = None, groups: int = 1,
               kept_groups: Optional[int] = None, group_top: int = 2, renormalize: bool = True,
               scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(weight, index)``, both ``[..., k]``: the ``k`` best experts of every row of ``logits[..., E]`` and their weights.

    ``s`` is ``softmax(logits)`` or ``sigmoid(logits)`` over the last dimension, in fp32.  The choice goes by ``s + bias``
    (``bias``: float32 ``[E]``, as a load-balancing rule updates it; it has no part in the weights and no gradient),
    largest first, ties to the lower index.  With ``groups`` above 1 the experts are that many equal groups of neighbours;
    only the ``kept_groups`` best groups are chosen from, a group's rank being the sum of its ``group_top`` (1 or 2) best
    ``s + bias``.  ``weight`` is ``s`` of the chosen experts, divided by its sum over them when ``renormalize``, times
    ``scale``, in the dtype of ``logits`` and differentiable (``index``, int64, is not; second derivatives are not built).

    An expert whose logit is ``-inf`` is masked: it comes after every other of the open groups and weighs 0; a row of
    nothing else has weights 0.  A NaN ranks with the masked ones and shows as NaN weights; under softmax a NaN or ``+inf``
    makes the whole row NaN, as with ``torch.softmax``, and its gradient.  The choice does not depend on how scores round: it compares the
    logits where the scores order as they do, and scores in 64 bits where a bias or a sum of two decides.

    The call can be captured into a graph; a backward pass together with its forward pass, on leaves that no other living
    autograd graph uses.

    float16, float32 and bfloat16 on a CUDA device; at most 1024 experts, 32 chosen, 32 groups.  Raises ``TypeError`` /
    ``ValueError`` for bad arguments and ``RuntimeError`` for tensors that are not on a CUDA device.
    """
    if not isinstance(logits, torch.Tensor):
        raise TypeError(f"logits must be a torch.Tensor, got {type(logits).__name__}")
    if logits.dim() < 1:
        raise ValueError("logits must have at least one dimension")
    if logits.dtype not in _SUPPORTED_DTYPES:
        raise TypeError(f"logits dtype must be one of float16, float32, bfloat16; got {logits.dtype}")
    if score not in _SCORES:
        raise ValueError(f"score must be 'softmax' or 'sigmoid', got {score!r}")
    experts = logits.size(-1)
    _check_int("the number of experts (logits.size(-1))", experts, 1, MAX_EXPERTS)
    _check_int("groups", groups, 1, min(MAX_GROUPS, experts))
    if experts % groups:
        raise ValueError(f"groups ({groups}) must divide the number of experts ({experts})")
    size = experts // groups
    if kept_groups is None:
        kept_groups = groups
    _check_int("kept_groups", kept_groups, 1, groups)
    _check_int("group_top", group_top, 1, 2)
    if groups == 1:
        group_top = 1
    elif group_top > size:
        raise ValueError(f"group_top ({group_top}) exceeds the size of a group ({size})")
    _check_int("k", k, 1, min(MAX_CHOSEN, size * kept_groups))
    if bias is not None:
        if not isinstance(bias, torch.Tensor):
            raise TypeError(f"bias must be a torch.Tensor, got {type(bias).__name__}")
        if bias.dtype != torch.float32:
            raise TypeError(f"bias dtype must be float32, got {bias.dtype}")
        if bias.dim() != 1 or bias.size(0) != experts:
            raise ValueError(f"bias must be 1-D with one value per expert ({experts}), got {tuple(bias.shape)}")
        if bias.device != logits.device:
            raise ValueError(f"logits and bias must be on the same device, got {logits.device} and {bias.device}")
        bias = bias.detach().contiguous()
    if logits.device.type != "cuda":
        raise RuntimeError("topk_route requires CUDA tensors")
    rows = logits if logits.dim() == 2 else logits.reshape(-1, experts)
    weight, index = _pybind.topk_route(rows.contiguous(), bias, k, _SCORES[score], groups, kept_groups, group_top, bool(renormalize),
                                       float(scale))
    if logits.dim() == 2:
        return weight, index
    shape = logits.shape[:-1] + (k,)
    return weight.view(shape), index.view(shape)
