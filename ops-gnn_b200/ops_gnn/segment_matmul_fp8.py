"""Segment products of block-scaled 8-bit values.  An addition: the reference has no counterpart."""
from typing import Optional

import torch

from . import _pybind
from .segment_matmul import check_segments

_OUT_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
BLOCK = 128


def segment_matmul_fp8(src: torch.Tensor, src_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                       indptr: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``out[r, n] = sum_k src[r, k] * src_scale[r, k // 128] * weight[e, n, k] * weight_scale[e, n // 128, k // 128]`` for the
    rows ``indptr[e] <= r < indptr[e + 1]`` of each segment ``e``.

    ``src`` is ``[M, K]`` and ``weight`` ``[E, N, K]``, both float8_e4m3fn; the scales are float32, ``[M, ceil(K / 128)]`` and
    ``[E, ceil(N / 128), ceil(K / 128)]``, any positive values (``quantize_fp8`` makes powers of two) whose products
    are within float32's range (the two scales of a block are multiplied first).  Without ``indptr``
    it is one dense product with ``weight`` ``[N, K]`` and ``weight_scale`` ``[ceil(N / 128), ceil(K / 128)]``.  The result
    ``[M, N]`` is ``out_dtype`` (bfloat16, float16 or float32).  Products of a block of 128 are added up on the tensor cores,
    blocks in fp32 registers, so no sum is held in fewer than 32 bits.

    Rows of no segment give 0; pointers are treated as in ``segment_matmul`` and stay on the device.  No autograd.  Raises
    ``TypeError`` / ``ValueError`` for bad arguments and ``RuntimeError`` for tensors that are not on a CUDA device.
    """
    for name, tensor, dtype in (("src", src, torch.float8_e4m3fn), ("weight", weight, torch.float8_e4m3fn),
                                ("src_scale", src_scale, torch.float32), ("weight_scale", weight_scale, torch.float32)):
        if not isinstance(tensor, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(tensor).__name__}")
        if tensor.dtype != dtype:
            raise TypeError(f"{name} dtype must be {dtype}, got {tensor.dtype}")
        if tensor.device != src.device:
            raise ValueError(f"src and {name} must be on the same device, got {src.device} and {tensor.device}")
    if out_dtype not in _OUT_DTYPES:
        raise TypeError(f"out_dtype must be one of float16, float32, bfloat16; got {out_dtype}")
    if src.dim() != 2:
        raise ValueError(f"src must be 2-D, got {src.dim()}-D")
    dims = 2 if indptr is None else 3
    if weight.dim() != dims or weight_scale.dim() != dims:
        raise ValueError(f"weight and weight_scale must be {dims}-D, got {weight.dim()}-D and {weight_scale.dim()}-D")
    if indptr is None:
        weight, weight_scale = weight.unsqueeze(0), weight_scale.unsqueeze(0)
    else:
        indptr = check_segments(src, indptr, weight.size(0))
    if weight.size(2) != src.size(1):
        raise ValueError(f"weight.size(-1) ({weight.size(2)}) must match src.size(1) ({src.size(1)})")
    blocks = -(-src.size(1) // BLOCK)
    if tuple(src_scale.shape) != (src.size(0), blocks):
        raise ValueError(f"src_scale must be {(src.size(0), blocks)}, got {tuple(src_scale.shape)}")
    want = (weight.size(0), -(-weight.size(1) // BLOCK), blocks)
    if tuple(weight_scale.shape) != want:
        raise ValueError(f"weight_scale must be {want if indptr is not None else want[1:]}, got "
                         f"{tuple(weight_scale.shape) if indptr is not None else tuple(weight_scale.shape[1:])}")
    if src.device.type != "cuda":
        raise RuntimeError("segment_matmul_fp8 requires CUDA tensors")
    return _pybind.segment_matmul_fp8(src, src_scale, weight, weight_scale, indptr, _OUT_DTYPES[out_dtype])
