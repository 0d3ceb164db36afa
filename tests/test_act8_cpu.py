"""CPU: what the 8-bit activations and the norms around a block refuse, before anything is launched."""

import pytest
import torch

from hackaton_b200 import Act8, act8_quantize, lora_grad_act8, sandwich_norm


def test_act8_refusals():
    with pytest.raises(TypeError, match="fp16, bf16 or fp32"):
        act8_quantize(torch.zeros(2, 32, dtype=torch.float64))
    with pytest.raises(ValueError, match="CUDA"):
        act8_quantize(torch.zeros(2, 32))
    kept = Act8(torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.uint8), (2, 32), torch.bfloat16)
    with pytest.raises(TypeError, match="fp16"):
        lora_grad_act8(kept, torch.zeros(2, 16, dtype=torch.float16))
    kept = Act8(kept.codes, kept.steps, (2, 32), torch.float16)
    with pytest.raises(TypeError, match="fp16"):
        lora_grad_act8(kept, torch.zeros(2, 16))
    for shape in ((3, 16), (2, 8), (4, 8)):
        with pytest.raises(ValueError):
            lora_grad_act8(kept, torch.zeros(shape, dtype=torch.float16))


def _sandwich(**change):
    args = dict(residual=torch.zeros(4, 8), delta=torch.zeros(4, 8, dtype=torch.float16), post_weight=torch.ones(8),
                pre_weight=torch.ones(8), eps=1e-6)
    args.update(change)
    return sandwich_norm(**args)


def test_sandwich_norm_needs_cuda():
    with pytest.raises(ValueError, match="CUDA"):
        _sandwich()


def test_sandwich_norm_refusals(monkeypatch):
    """The checks behind the one for the device, on tensors that only claim to be on it."""
    from hackaton_b200 import sandwich

    def check(**change):
        class Claimed:
            def __init__(self, t):
                self.t, self.is_cuda, self.device = t, True, "cuda:0"
                self.dtype, self.shape = t.dtype, t.shape

            def dim(self):
                return self.t.dim()

        args = dict(residual=torch.zeros(4, 8), delta=torch.zeros(4, 8, dtype=torch.float16), post_weight=torch.ones(8),
                    pre_weight=torch.ones(8), gate=None, out_dtype=torch.float16)
        args.update(change)
        sandwich._validate(*[Claimed(v) if isinstance(v, torch.Tensor) else v for v in args.values()])

    check()
    check(out_dtype=torch.float32)
    for change in (dict(residual=torch.zeros(4, 8).half()), dict(post_weight=torch.ones(8).half()),
                   dict(delta=torch.zeros(4, 8, dtype=torch.float64)), dict(out_dtype=torch.bfloat16),
                   dict(gate=torch.ones(8).half())):
        with pytest.raises(TypeError):
            check(**change)
    for change in (dict(delta=torch.zeros(4, 9).half()), dict(post_weight=torch.ones(7)), dict(pre_weight=torch.ones(1, 8)),
                   dict(residual=torch.zeros(4, 16385), delta=torch.zeros(4, 16385).half(),
                        post_weight=torch.ones(16385), pre_weight=torch.ones(16385))):
        with pytest.raises(ValueError):
            check(**change)


@pytest.mark.parametrize("gate,stream,rows", [((8,), (6, 8), 1), ((1, 8), (6, 8), 1), ((3, 8), (6, 8), 3), ((6, 8), (6, 8), 6),
                                              ((2, 1, 8), (2, 5, 8), 2), ((2, 5, 8), (2, 5, 8), 10), ((1, 1, 8), (2, 5, 8), 1),
                                              ((8,), (2, 5, 8), 1), ((8,), (8,), 1), ((2, 3, 1, 8), (2, 3, 4, 8), 6)])
def test_gate_shapes(gate, stream, rows):
    from hackaton_b200.sandwich import _gate_rows

    assert _gate_rows(torch.ones(gate), stream).shape == (rows, 8)


@pytest.mark.parametrize("gate,stream", [((4, 8), (6, 8)), ((7,), (6, 8)), ((5, 8), (2, 5, 8)), ((1, 5, 8), (2, 5, 8)),
                                         ((2, 8), (2, 5, 8)), ((12, 8), (6, 8)), ((2, 1, 4, 8), (2, 3, 4, 8)), ((6, 1), (6, 8))])
def test_gate_shapes_that_do_not_run_over_consecutive_rows(gate, stream):
    from hackaton_b200.sandwich import _gate_rows

    with pytest.raises(ValueError, match="gate"):
        _gate_rows(torch.ones(gate), stream)
