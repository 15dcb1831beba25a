"""The CSR structure of (row, expert) pairs.  An addition: the reference has no counterpart."""
from typing import Tuple

import torch

from . import _pybind

MAX_EXPERTS = 4096


def route_csr(index: torch.Tensor, num_experts: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(indptr, perm, position)`` of expert labels, all int64 on the device of ``index``.

    ``index`` (int32 / int64, any shape, for instance ``[T, k]`` from ``topk_route``) holds one label per pair; the pairs
    are numbered as they lie in memory.  ``perm`` lists the pairs expert by expert, those of one expert in their own order
    (a stable sort); expert ``e`` owns ``perm[indptr[e]:indptr[e + 1]]``; ``position``, of the shape of ``index``, is where
    each pair went (``perm[position] = 0, 1, 2, ...``).  A label outside ``[0, num_experts)`` is a dropped pair: those come
    last, behind ``indptr[num_experts]``, where ``segment_matmul`` gives 0.  Nothing is read back to the host.

    A layer of experts over rows ``x`` with ``weight, index = topk_route(...)``::

        indptr, perm, position = route_csr(index, E)
        y = segment_matmul(x[perm // k], indptr, w)                     # each pair's row through its expert
        out = (y[position] * weight.unsqueeze(-1)).sum(1)               # or csr_spmm over position and weight

    At most 4096 experts and 2^31 - 1 pairs.  Raises ``TypeError`` / ``ValueError`` for bad arguments and ``RuntimeError``
    for tensors that are not on a CUDA device.
    """
    if not isinstance(index, torch.Tensor):
        raise TypeError(f"index must be a torch.Tensor, got {type(index).__name__}")
    if index.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"index dtype must be int32 or int64, got {index.dtype}")
    if not isinstance(num_experts, int) or isinstance(num_experts, bool):
        raise TypeError(f"num_experts must be an int, got {type(num_experts).__name__}")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"num_experts must be in [1, {MAX_EXPERTS}], got {num_experts}")
    if index.numel() >= 2 ** 31:
        raise ValueError(f"index must hold fewer than 2^31 labels, got {index.numel()}")
    if index.device.type != "cuda":
        raise RuntimeError("route_csr requires CUDA tensors")
    return _pybind.route_csr(index.contiguous(), num_experts)
