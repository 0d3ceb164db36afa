"""CPU: what the vocabulary loss and the activations kept in 8 bits refuse, before anything is launched."""

import pytest
import torch

from hackaton_b200 import act8_dequantize, silu_mul, vocab_cross_entropy
from hackaton_b200.act8 import Act8


def test_vocab_cross_entropy_needs_cuda():
    with pytest.raises(ValueError, match="CUDA"):
        vocab_cross_entropy(torch.zeros(2, 8).half(), torch.zeros(5, 8).half(), torch.zeros(2, dtype=torch.int64))


def test_vocab_cross_entropy_refusals():
    """The checks behind the one for the device, on tensors that only claim to be on it."""
    from hackaton_b200 import lm_loss

    class Claimed:
        def __init__(self, t, device="cuda:0"):
            self.is_cuda, self.device, self.dtype, self.shape, self.t = True, device, t.dtype, t.shape, t

        def dim(self):
            return self.t.dim()

    def check(h, w, t, device="cuda:0"):
        lm_loss._refuse_vocab(Claimed(h), Claimed(w), Claimed(t, device))

    half = lambda *s: torch.zeros(s, dtype=torch.float16)
    index = lambda *s: torch.zeros(s, dtype=torch.int64)
    for h, w, t in ((half(2, 8), half(5, 8).bfloat16(), index(2)), (half(2, 8).float(), half(5, 8).float(), index(2)),
                    (half(2, 8), half(5, 8), index(2).int())):
        with pytest.raises(TypeError):
            check(h, w, t)
    for h, w, t in ((half(2, 8), half(5, 16), index(2)), (half(2, 8), half(5, 8), index(3)), (half(2, 8), half(5, 1, 8), index(2)),
                    (half(2, 3, 8), half(5, 8), index(6)), (half(2, 12), half(5, 12), index(2)), (half(2, 8), half(0, 8), index(2)),
                    (half(2, 0), half(5, 0), index(2)), (half(), half(5, 8), index())):
        with pytest.raises(ValueError):
            check(h, w, t)
    with pytest.raises(ValueError, match="devices"):
        check(half(2, 8), half(5, 8), index(2), "cuda:1")


def test_kept_swiglu_refusals():
    with pytest.raises(ValueError, match="CUDA"):
        silu_mul(torch.zeros(2, 8).half().requires_grad_(), torch.zeros(2, 8).half(), keep8=True)
    with pytest.raises(ValueError, match="CUDA"):
        act8_dequantize(Act8(torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.uint8), (2, 32), torch.float16))
