"""What candidate_loss refuses, without a GPU (its checks run before any kernel)."""
import pytest
import torch

from unicorn_amd.candidates import candidate_loss
from unicorn_amd.routing import Routing


def test_refusals():
    r = Routing(torch.full((3, 2), 0.5), torch.tensor([[0, 1]] * 3), torch.tensor([3, 3, 0], dtype=torch.int32))
    errors, scores = torch.rand(3, 2), torch.randn(3, 3)
    for temperature in (0.0, -0.1, float("nan")):
        with pytest.raises(ValueError, match="temperature must be positive"):
            candidate_loss(errors, r, scores, temperature=temperature)
    for bad in (errors[:, 0], errors[:, :1], errors[0], errors.t()):
        with pytest.raises(ValueError, match="errors must have shape"):
            candidate_loss(bad, r, scores)
