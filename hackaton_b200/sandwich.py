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
from ._autograd import call

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


def _launch(op, residual, delta, post_weight, pre_weight, gate, train):
    hidden = residual.shape[-1]
    r2, d2 = residual.reshape(-1, hidden).contiguous(), delta.reshape(-1, hidden).contiguous()
    post, pre = post_weight.contiguous(), pre_weight.contiguous()
    g2 = None if gate is None or r2.shape[0] == 0 else _gate_rows(gate, residual.shape)
    stream, normed, rstd = _lib.host().sandwich_fwd(r2, d2, post, pre, g2, op.scale, op.eps,
                                                    op.out_dtype == torch.float32, train)
    return stream, normed, rstd, (d2, post, pre, g2)


class _SandwichOp:
    def __init__(self, eps, scale, out_dtype):
        self.eps, self.scale, self.out_dtype = eps, scale, out_dtype

    def run(self, keep, residual, delta, post_weight, pre_weight, gate):
        stream, normed, rstd, read = _launch(self, residual, delta, post_weight, pre_weight, gate, True)
        keep(stream, *read, rstd, shape=residual.shape, gate_shape=None if gate is None else gate.shape)
        return stream.reshape(residual.shape), normed.reshape(residual.shape)

    def grad(self, kept, d_stream, d_normed):
        stream, d2, post, pre, g2, rstd = kept.tensors
        grads = _lib.host().sandwich_bwd(stream, d2, post, pre, g2, rstd,
                                         d_stream.reshape(stream.shape).float().contiguous(),
                                         d_normed.reshape(stream.shape).contiguous(), self.scale, list(kept.wants))
        shapes = [kept.shape, kept.shape, post.shape, pre.shape, kept.gate_shape]
        out = [None if g is None else g.reshape(shape) for g, shape in zip(grads, shapes)]
        if kept.gate_shape is not None and g2 is None and kept.wants[4]:     # (no rows)
            out[4] = torch.zeros(kept.gate_shape, dtype=torch.float32, device=stream.device)
        return tuple(out)


def sandwich_norm(residual, delta, post_weight, pre_weight, eps, gate=None, residual_scale=1.0, out_dtype=None):
    """(stream, normed) as above. residual: fp32 [..., hidden]; delta: the block's output, fp16, bf16 or fp32 of the same
    shape; post_weight, pre_weight: fp32 [hidden]; gate: None, or fp32 [hidden], or leading dimensions of the stream's
    followed by ones ([batch, 1, hidden] over [batch, tokens, hidden]), or [gates, hidden] over [rows, hidden] with row g
    for the g-th share of consecutive rows; residual_scale: a number; out_dtype of `normed`: delta's type (the default)
    or fp32. Gradients flow to all five tensors."""
    out_dtype = delta.dtype if out_dtype is None else out_dtype
    _validate(residual, delta, post_weight, pre_weight, gate, out_dtype)
    if gate is not None and residual.numel() > 0:
        _gate_rows(gate, residual.shape)
    op = _SandwichOp(float(eps), float(residual_scale), out_dtype)
    tensors = (residual, delta, post_weight, pre_weight, gate)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return call(op, *tensors)
    stream, normed, *_ = _launch(op, *tensors, False)
    return stream.reshape(residual.shape), normed.reshape(residual.shape)
