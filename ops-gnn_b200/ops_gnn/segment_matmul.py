"""One matrix product per CSR segment.  An addition: the reference has no counterpart; its segment operators reduce rows,
this one multiplies them (typed linear layers of relational graphs, experts of a routed layer)."""
import torch

from . import _pybind

_SUPPORTED_DTYPES = (torch.float16, torch.float32, torch.bfloat16)
_SUPPORTED_PTR_DTYPES = (torch.int32, torch.int64)


def check_segments(src: torch.Tensor, indptr: torch.Tensor, segments: int) -> torch.Tensor:
    if not isinstance(indptr, torch.Tensor):
        raise TypeError(f"indptr must be a torch.Tensor, got {type(indptr).__name__}")
    if indptr.dtype not in _SUPPORTED_PTR_DTYPES:
        raise TypeError(f"indptr dtype must be int32 or int64, got {indptr.dtype}")
    if indptr.dim() != 1:
        raise ValueError(f"indptr must be 1-D, got {indptr.dim()}-D")
    if indptr.numel() != segments + 1:
        raise ValueError(f"indptr must hold one pointer more than weight has matrices ({segments}), got {indptr.numel()}")
    if indptr.device != src.device:
        raise ValueError(f"src and indptr must be on the same device, got {src.device} and {indptr.device}")
    return indptr.contiguous()


def segment_matmul(src: torch.Tensor, indptr: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """``out[r] = src[r] @ weight[e]`` for the rows ``indptr[e] <= r < indptr[e + 1]`` of each segment ``e``.

    ``src`` is ``[M, K]``, ``weight`` ``[E, K, N]`` of the same dtype (float16, float32 or bfloat16), ``indptr`` ``[E + 1]``
    (int32 / int64, non-decreasing); the result is ``[M, N]``.  Segments may be empty; rows before ``indptr[0]`` and from
    ``indptr[E]`` on belong to none and give 0, and have gradient 0.  Sums are held in fp32 and rounded once.  Any strides:
    rows of ``src`` and either layout of ``weight`` (``weight.transpose(1, 2)`` of ``[E, N, K]``) are read in place, other
    layouts are copied first.  Differentiable in ``src`` and ``weight`` (second derivatives are not built).

    Larger float32 products take scratch memory of about 1.5 times their operands while they run; their values below 2^-110
    lose low bits, and an infinity or a value above 3.389e38 among the operands makes them several times slower (a NaN does not).
    16-bit operands whose rows are off 16-byte boundaries are copied onto them where that pays.  Every sum is taken in a fixed order: the same call gives the same bits.

    The pointers stay on the device: nothing is read back, so the call can be captured into a graph and replayed with other
    pointers.  (A backward pass is captured together with its forward pass, on leaves that no other living autograd graph uses:
    torch joins the streams of all of a leaf's uses.)  A pointer outside ``[0, M]`` counts as the nearer end.  Their order is not checked: where they descend, rows
    and gradients of the segments concerned are unspecified, but nothing outside the tensors is read or written.  Raises
    ``TypeError`` / ``ValueError`` for bad arguments and ``RuntimeError`` for tensors that are not on a CUDA device.
    """
    if not isinstance(src, torch.Tensor):
        raise TypeError(f"src must be a torch.Tensor, got {type(src).__name__}")
    if not isinstance(weight, torch.Tensor):
        raise TypeError(f"weight must be a torch.Tensor, got {type(weight).__name__}")
    if src.dtype not in _SUPPORTED_DTYPES:
        raise TypeError(f"src dtype must be one of float16, float32, bfloat16; got {src.dtype}")
    if weight.dtype != src.dtype:
        raise TypeError(f"weight dtype must match src ({src.dtype}), got {weight.dtype}")
    if src.dim() != 2:
        raise ValueError(f"src must be 2-D, got {src.dim()}-D")
    if weight.dim() != 3:
        raise ValueError(f"weight must be 3-D, got {weight.dim()}-D")
    if weight.size(1) != src.size(1):
        raise ValueError(f"weight.size(1) ({weight.size(1)}) must match src.size(1) ({src.size(1)})")
    if weight.device != src.device:
        raise ValueError(f"src and weight must be on the same device, got {src.device} and {weight.device}")
    indptr = check_segments(src, indptr, weight.size(0))
    if src.device.type != "cuda":
        raise RuntimeError("segment_matmul requires CUDA tensors")
    return _pybind.segment_matmul(src, indptr, weight)
