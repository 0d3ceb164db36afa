"""CPU: what the operators around a training step refuse before anything else is looked at."""

import pytest
import torch

from hackaton_b200 import sandwich_norm


def test_sandwich_norm_refuses_a_scale_that_wants_a_gradient():
    """It would get none, and nobody would tell."""
    ones = torch.ones(8)
    with pytest.raises(TypeError, match="residual_scale"):
        sandwich_norm(torch.zeros(4, 8), torch.zeros(4, 8).half(), ones, ones, 1e-6, residual_scale=torch.ones((), requires_grad=True))
    with pytest.raises(ValueError, match="CUDA"):       # a number in a tensor is one
        sandwich_norm(torch.zeros(4, 8), torch.zeros(4, 8).half(), ones, ones, 1e-6, residual_scale=torch.ones(()))
