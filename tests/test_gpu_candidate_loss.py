"""candidate_loss with empty slots: whatever error stands there, neither the loss nor a gradient takes it up."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 1e30])
def test_errors_of_empty_slots_are_left_out(bad):
    from unicorn_amd.candidates import candidate_loss
    from unicorn_amd.routing import route_candidates
    scores = torch.randn(4, 5, generator=torch.Generator().manual_seed(1)).cuda()
    scores[1, 1:], scores[2] = -float("inf"), -float("inf")
    results = []
    for value in (0.25, bad):
        x = scores.clone().requires_grad_(True)
        r = route_candidates(x, 3)
        errors = torch.rand(4, 3, generator=torch.Generator().manual_seed(2)).cuda()
        errors = torch.where(r.indices < 0, value, errors).requires_grad_(True)
        loss = candidate_loss(errors, r, x, temperature=0.1)
        results.append((loss.detach(),) + torch.autograd.grad(loss.sum(), (x, errors)))
    assert int((r.indices < 0).sum()) == 2 + 3
    for a, b in zip(*results):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, b)
    assert bool((results[1][2][r.indices < 0] == 0).all()) and float(results[1][0][2]) == 0.0
