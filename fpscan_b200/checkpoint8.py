"""Activation checkpoints in 8 bits.

What a recurrence keeps for its backward pass can be kept in 8 bits:

* ``quantize8(x)`` -> ``(codes, steps)`` and ``dequantize8(codes, steps, dtype)``: a tensor in blocks of
  64 consecutive values, each block with one fp32 step;
* ``pscan_channels_last(..., checkpoint8=True)`` (ops.py) keeps its output so, inside the scan kernels;
* ``gated_delta(..., checkpoint8=True)`` (delta.py) keeps q, k and v so.

A block's step is its largest magnitude over 127 and a value becomes the nearest multiple of it (ties to
even), so it is off by at most half a step, 1/254 of the block's largest magnitude, before it is rounded to
the type it is read back in (steps are fp32 numbers: magnitudes below 2^-119 are off by up to 2^-143
besides).  A block that holds an infinity or a NaN reads back as NaN.  The reference saves its tensors as they are (fpscan/ops.py:64-67).
"""
from __future__ import annotations

from typing import Tuple

import torch

from .ops import _EXT, DTYPE_CODES, _check_input, _launch

__all__ = ["quantize8", "dequantize8"]

BLOCK = 64


def quantize8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x`` (contiguous, float32 / float16 / bfloat16, any shape) in 8 bits: int8 codes of x's shape and
    fp32 steps, one per 64 consecutive values.  No autograd."""
    if _EXT is not None and isinstance(x, torch.Tensor):
        return _EXT.quantize8(x)
    _check_input(x, "x")
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    steps = torch.empty((x.numel() + BLOCK - 1) // BLOCK, dtype=torch.float32, device=x.device)
    if x.numel():
        _launch(x.get_device(), "fpscan_quantize8", x.data_ptr(), codes.data_ptr(), steps.data_ptr(),
                x.numel(), DTYPE_CODES[x.dtype])
    return codes, steps


def dequantize8(codes: torch.Tensor, steps: torch.Tensor,
                dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that ``quantize8``'s result stands for, rounded to ``dtype``."""
    for t, name, want in ((codes, "codes", torch.int8), (steps, "steps", torch.float32)):
        if not isinstance(t, torch.Tensor):
            raise RuntimeError(f"{name} must be a torch.Tensor")
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor")
        if not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous")
        if t.dtype != want:
            raise RuntimeError(f"{name} must be {want} (got {t.dtype})")
    if dtype not in DTYPE_CODES:
        raise RuntimeError(f"dtype must be float16 or bfloat16 or float32 (got {dtype})")
    if codes.device != steps.device:
        raise RuntimeError("codes and steps must be on the same device")
    n = codes.numel()
    if steps.numel() != (n + BLOCK - 1) // BLOCK:
        raise RuntimeError(f"steps must hold one value per {BLOCK} codes: {(n + BLOCK - 1) // BLOCK}, "
                           f"got {steps.numel()}")
    if _EXT is not None:
        return _EXT.dequantize8(codes, steps, dtype)
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    if n:
        _launch(codes.get_device(), "fpscan_dequantize8", codes.data_ptr(), steps.data_ptr(),
                out.data_ptr(), n, DTYPE_CODES[dtype])
    return out
