"""Activations kept in 8 bits for the backward pass, and their use there.

What a training step keeps of a block between its two directions is mostly 16-bit activations: the input of each
LoRA linear (for the gradient of its first factor), gate and up of each MLP (for the SwiGLU backward). Here they are
kept as int8 codes with one power of two per 32 values of a row, 1.03 bytes a value; nothing else of the forward or
the backward changes. The reference moves such tensors to host memory instead (solution/kernels.py:60-91).

    step = 2^e, e = floor(log2 max|x|) - 6;  code = rint(x / step) within -127 .. 127;  value = code * step

A value is off by at most 2^-7 of the largest of its 32, half that below 127.5 / 128 of it. The arithmetic is exact
apart from the rounding to a whole code: the values do not depend on how they are computed. A block that holds an
infinity or a NaN is read back as NaN, so that what watches gradients for them still sees them.

Users: `silu_mul(..., keep8=True)`, `nf4_swiglu_mlp(..., keep8=True)`, `nf4_lora_linear(..., keep8=True)`,
`nf4_linear_group(..., keep8=True)`.
"""

from __future__ import annotations

import torch

from . import _lib

BLOCK = 32     # values of a row that share a step
RANK = 16
_TYPES = (torch.float16, torch.bfloat16, torch.float32)
_LIKE = {t: torch.empty(0, dtype=t) for t in _TYPES}


class Act8:
    """A tensor of `shape` and `dtype` in 8 bits: codes int8 [rows, ceil(cols / 32) * 32], steps uint8
    [rows, ceil(cols / 32)]."""

    __slots__ = ("codes", "steps", "shape", "dtype")

    def __init__(self, codes, steps, shape, dtype):
        self.codes, self.steps, self.shape, self.dtype = codes, steps, shape, dtype

    def __repr__(self):
        return f"Act8({tuple(self.shape)}, {self.dtype}, {self.codes.device})"

    @property
    def nbytes(self):
        return self.codes.numel() + self.steps.numel()


def act8_quantize(x):
    """`x` (fp16, bf16 or fp32, CUDA, at least one dimension) in 8 bits; blocks run along the last dimension. No gradient
    leads back from the parts to `x` (it is what a backward pass keeps); a tangent of forward mode is refused."""
    kept = _lib.host().act8_quantize(x)
    if kept is None:
        if x.dtype not in _TYPES:
            raise TypeError(f"hackaton_b200: activations are kept from fp16, bf16 or fp32, got {x.dtype}")
        if not x.is_cuda:
            raise ValueError("hackaton_b200: act8_quantize needs a CUDA tensor (there is no CPU path)")
        raise ValueError("hackaton_b200: act8_quantize needs at least one dimension")
    return Act8(*kept, x.shape, x.dtype)


def _refuse_parts(kept):
    if not (kept.codes.is_cuda and kept.steps.is_cuda):
        raise ValueError("hackaton_b200: activations in 8 bits need CUDA tensors (there is no CPU path)")
    raise ValueError(f"hackaton_b200: codes {tuple(kept.codes.shape)} {kept.codes.dtype} and steps {tuple(kept.steps.shape)} "
                     f"{kept.steps.dtype} are not a tensor of shape {tuple(kept.shape)} as act8_quantize makes it")


def act8_dequantize(kept):
    """The values that `kept` holds, in the shape and type it was made from."""
    if kept.dtype not in _TYPES:
        raise TypeError(f"hackaton_b200: activations are kept from fp16, bf16 or fp32, got {kept.dtype}")
    values = _lib.host().act8_dequantize(kept.codes, kept.steps, kept.shape, _LIKE[kept.dtype])
    if values is None:
        _refuse_parts(kept)
    return values


def lora_grad_act8(kept, s):
    """sᵀ . x as fp32 [16, cols] for an fp16 input x kept in 8 bits and fp16 s [..., 16] with a row for each of
    its rows: the gradient of a LoRA pair's first factor (`lora.lora_grad` with rank-major output), in a fixed
    order of additions. As a part of backward passes it has no gradient of its own."""
    grad = _lib.host().act8_lora_grad(kept.codes, kept.steps, s, kept.shape[-1]) if kept.dtype is torch.float16 else None
    if grad is None:
        if kept.dtype != torch.float16 or s.dtype != torch.float16:
            raise TypeError(f"hackaton_b200: the LoRA gradient computes from fp16, got {kept.dtype} and {s.dtype}")
        if s.device != kept.codes.device:
            raise ValueError(f"hackaton_b200: operands on {kept.codes.device} and {s.device}")
        if s.dim() == 0 or s.shape[-1] != 16 or s.numel() != kept.codes.shape[0] * 16:
            raise ValueError(f"hackaton_b200: {tuple(s.shape)} for an input of shape {tuple(kept.shape)}")
        _refuse_parts(kept)
    return grad
