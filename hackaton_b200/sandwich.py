"""The norms around a block, its gate and the residual in one pass each way, on the fp32 stream:

    n      = RMSNorm(delta) * post_weight              the norm behind the block
    stream = residual_scale * residual + gate * n      its gate (layer scale, or a row per sequence), the residual
    normed = RMSNorm(stream) * pre_weight              the norm before the next block, in the projections' type

`rmsnorm.add_rms_norm` is the same step without the first norm, gate and scale. Next to the inputs two fp32 numbers per row
are kept for the gradient pass, which is one kernel and a small one that adds up the weights' column sums.
"""

from __future__ import annotations

import torch

from . import _lib

MAX_HIDDEN = 16384


def _gate_rows(gate, shape):
    """Rows of the gate, each for as many consecutive rows of the stream; the shapes it may have are those that
    broadcast to the stream's in that way."""
    hidden = shape[-1]
    if gate.dim() == 0 or gate.shape[-1] != hidden:
        raise ValueError(f"hackaton_b200: gate {tuple(gate.shape)} for a stream of {tuple(shape)}")
    lead = tuple(gate.shape[:-1])
    rows = 1
    for n in shape[:-1]:
        rows *= n
    count = gate.numel() // hidden
    if len(shape) == 2 and len(lead) == 1:     # [gates, hidden] over packed rows
        fits = count > 0 and rows % count == 0
    else:                                      # leading dimensions of the stream's, ones behind them
        k = 0
        while k < len(lead) and lead[k] == shape[k] and k < len(shape) - 1:
            k += 1
        fits = all(n == 1 for n in lead) or (len(lead) == len(shape) - 1 and all(n == 1 for n in lead[k:]))
    if not fits:
        raise ValueError(f"hackaton_b200: gate {tuple(gate.shape)} for a stream of {tuple(shape)}: [hidden], the "
                         "stream's leading dimensions followed by ones, or [gates, hidden] over [rows, hidden]")
    return gate.reshape(count, hidden).contiguous()


def _validate(residual, delta, post_weight, pre_weight, gate, out_dtype):
    tensors = [residual, delta, post_weight, pre_weight] + ([] if gate is None else [gate])
    if not all(t.is_cuda for t in tensors):
        raise ValueError("hackaton_b200: sandwich_norm needs CUDA tensors (there is no CPU path)")
    if any(t.device != residual.device for t in tensors):
        raise ValueError("hackaton_b200: sandwich_norm: tensors on different devices")
    if residual.dtype != torch.float32 or any(t.dtype != torch.float32 for t in tensors[2:]):
        raise TypeError("hackaton_b200: sandwich_norm: stream, weights and gate are fp32, got "
                        + ", ".join(str(t.dtype) for t in tensors[:1] + tensors[2:]))
    if delta.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError(f"hackaton_b200: sandwich_norm: delta is fp16, bf16 or fp32, got {delta.dtype}")
    if out_dtype not in (delta.dtype, torch.float32):
        raise TypeError(f"hackaton_b200: sandwich_norm: the output is {delta.dtype} like delta or fp32, got {out_dtype}")
    if residual.dim() == 0 or delta.shape != residual.shape:
        raise ValueError(f"hackaton_b200: sandwich_norm adds a tensor of the residual's shape, got "
                         f"{tuple(delta.shape)} for {tuple(residual.shape)}")
    hidden = residual.shape[-1]
    if not 1 <= hidden <= MAX_HIDDEN:
        raise ValueError(f"hackaton_b200: sandwich_norm: rows of 1 to {MAX_HIDDEN} values, got {hidden}")
    if tuple(post_weight.shape) != (hidden,) or tuple(pre_weight.shape) != (hidden,):
        raise ValueError("hackaton_b200: sandwich_norm weights do not match the last dimension")


def sandwich_norm(residual, delta, post_weight, pre_weight, eps, gate=None, residual_scale=1.0, out_dtype=None):
    """(stream, normed) as above. residual: fp32 [..., hidden]; delta: the block's output, fp16, bf16 or fp32 of the same
    shape; post_weight, pre_weight: fp32 [hidden]; gate: None, or fp32 [hidden], or leading dimensions of the stream's
    followed by ones ([batch, 1, hidden] over [batch, tokens, hidden]), or [gates, hidden] over [rows, hidden] with row g
    for the g-th share of consecutive rows; residual_scale: a number (a tensor that requires a gradient is
    refused); out_dtype of `normed`: delta's type (the default)
    or fp32. Gradients flow to all five tensors, once
    and in reverse mode."""
    if isinstance(residual_scale, torch.Tensor) and residual_scale.requires_grad:
        raise TypeError("hackaton_b200: sandwich_norm: residual_scale is a number, no gradient flows to it; scale the residual before the call")
    given = gate
    if gate is not None and residual.dim() != 2 and gate.dim() > 1 and gate.shape[-1] == residual.shape[-1]:
        gate = _gate_rows(gate, residual.shape) if residual.numel() else gate.reshape(-1, gate.shape[-1])
    out = None
    if out_dtype is None or out_dtype in (delta.dtype, torch.float32):
        out = _lib.host().sandwich_norm(residual, delta, post_weight, pre_weight, gate, float(residual_scale), float(eps),
                                        out_dtype is torch.float32)
    if out is None:
        _validate(residual, delta, post_weight, pre_weight, given, delta.dtype if out_dtype is None else out_dtype)
        if given is not None:
            _gate_rows(given, residual.shape)
        raise ValueError("hackaton_b200: sandwich_norm does not take these tensors")
    return out
