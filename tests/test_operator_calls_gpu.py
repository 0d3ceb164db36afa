"""GPU: what the operators around a training step answer to calls beside the usual one."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from test_act8_gpu import activations

pytestmark = pytest.mark.gpu


def test_forward_mode_is_refused(cuda_lib):
    """A tangent is not dropped silently, with gradients on or off, whichever operand carries it."""
    from hackaton_b200 import act8_quantize, lora_grad_act8, sandwich_norm, silu_mul, vocab_cross_entropy

    x = activations(4, 64, torch.float16).clamp(-4, 4)
    s = activations(4, 16, torch.float16).clamp(-4, 4)
    ones, t = torch.ones(64, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    kept = act8_quantize(x)
    calls = [lambda d: vocab_cross_entropy(d(x), x, t), lambda d: vocab_cross_entropy(x, d(x), t),
             lambda d: sandwich_norm(d(x.float()), x, ones, ones, 1e-6), lambda d: sandwich_norm(x.float(), d(x), ones, ones, 1e-6),
             lambda d: sandwich_norm(x.float(), x, d(ones), ones, 1e-6), lambda d: sandwich_norm(x.float(), x, ones, d(ones), 1e-6),
             lambda d: sandwich_norm(x.float(), x, ones, ones, 1e-6, gate=d(ones)),
             lambda d: silu_mul(d(x), x, keep8=True), lambda d: silu_mul(x, d(x.clone().requires_grad_()), keep8=True),
             lambda d: act8_quantize(d(x)), lambda d: lora_grad_act8(kept, d(s))]
    with fwad.dual_level():
        dual = lambda v: fwad.make_dual(v, torch.ones_like(v))
        for call in calls:
            call(lambda v: v)
            with pytest.raises(RuntimeError):        # (NotImplementedError is one)
                call(dual)
            with torch.no_grad(), pytest.raises(RuntimeError):
                call(dual)
