"""Block-scaled 8-bit values.  An addition: the reference has no counterpart (its 8-bit type is int8 without scales)."""
from typing import Tuple

import torch

from . import _pybind

_SUPPORTED_DTYPES = (torch.float16, torch.float32, torch.bfloat16)
BLOCK = 128


def quantize_fp8(src: torch.Tensor, block_rows: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(values, scale)``: ``src[..., R, K]`` as float8_e4m3fn values of the same shape and one float32 scale per block.

    ``block_rows`` 1: a block is 128 consecutive columns of one row, ``scale`` is ``[..., R, ceil(K / 128)]`` (rows of
    activations).  ``block_rows`` 128: a block is a tile of 128 x 128, ``scale`` is ``[..., ceil(R / 128), ceil(K / 128)]``
    (weights).  The last block of a row or column may be short.  ``values * scale`` stands for ``src``.

    A scale is the smallest power of two that brings the largest finite magnitude of its block to at most 448, the largest
    float8_e4m3fn (never below 2^-126; 1 for a block of zeros), so the division is exact and each value is rounded once, to
    nearest, ties to even.  Infinities become 448 with their sign, NaN stays NaN.

    float16, float32 or bfloat16 on a CUDA device.  Raises ``TypeError`` / ``ValueError`` for bad arguments and
    ``RuntimeError`` for tensors that are not on a CUDA device.  No autograd.
    """
    if not isinstance(src, torch.Tensor):
        raise TypeError(f"src must be a torch.Tensor, got {type(src).__name__}")
    if src.dtype not in _SUPPORTED_DTYPES:
        raise TypeError(f"src dtype must be one of float16, float32, bfloat16; got {src.dtype}")
    if src.dim() < 2:
        raise ValueError(f"src must have at least two dimensions, got {src.dim()}")
    if not isinstance(block_rows, int) or isinstance(block_rows, bool):
        raise TypeError(f"block_rows must be an int, got {type(block_rows).__name__}")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"block_rows must be 1 or {BLOCK}, got {block_rows}")
    if src.device.type != "cuda":
        raise RuntimeError("quantize_fp8 requires CUDA tensors")
    return _pybind.quantize_fp8(src.contiguous(), block_rows)
