"""Candidate poses of a training step: predicted, chosen, rendered, and learnt from.

The reference predicts K candidate poses per image with a probability each, renders all K and weighs the losses by the
probabilities, kept apart by a balance loss (unicorn.py:295-304, 232-233).  Here the scores choose `top_k` of the K, only those are
rendered (`Renderer.render_candidates`), and the scores learn from the rendered candidates' errors:

    head = CandidateHead(latent, n_candidates=K, n_params=6)
    scores, params = head(z)                                         # (B, K), (B, K, 6)
    shown = renderer.render_candidates(meshes, R, T, scores, top_k=2, bias=bias)      # images (B, 2, 4, H, W), routing
    errors = ((shown.images[:, :, :3] - target[:, None]) ** 2).flatten(2).mean(2)     # (B, 2)
    loss = candidate_loss(errors, shown.routing, scores, temperature=0.01)            # (B,)
    update_balance_bias(bias, shown.routing.counts, 1e-3)
"""
from typing import NamedTuple

import torch
from torch import nn

from .distillation import distill_top_logits
from .normalization import LayerNorm
from .routing import Routing, update_balance_bias  # noqa: F401  (offered with the rest of the step)


class CandidateImages(NamedTuple):
    """What `Renderer.render_candidates` returns: images (B, k, 4, H, W) of the chosen candidates, and the choice."""
    images: torch.Tensor
    routing: Routing


class CandidateHead(nn.Module):
    """latent (B, D) -> scores (B, K) and parameters (B, K, P) of K candidates, from the normalised latent."""

    def __init__(self, dim, n_candidates, n_params):
        super().__init__()
        self.n_candidates, self.n_params = int(n_candidates), int(n_params)
        self.norm = LayerNorm(dim)
        self.score = nn.Linear(dim, self.n_candidates)
        self.params = nn.Linear(dim, self.n_candidates * self.n_params)

    def forward(self, z):
        z = self.norm(z)
        return self.score(z), self.params(z).view(z.shape[:-1] + (self.n_candidates, self.n_params))


def chosen_poses(R, T, routing):
    """Poses of the chosen candidates in the order `repeat` tiles meshes (image n shows mesh n % B): R (B,K,3,3) and
    T (B,K,3) -> (k*B,3,3), (k*B,3).  An empty slot takes candidate 0's pose; its weight is 0."""
    B, K = R.shape[:2]
    pick = routing.indices.clamp(min=0) + torch.arange(B, device=R.device)[:, None] * K
    pick = pick.t().reshape(-1)
    return R.reshape(B * K, 3, 3)[pick], T.reshape(B * K, 3)[pick]


def candidate_loss(errors, routing, scores, temperature=1.0, score_weight=1.0):
    """Per image (B,): the chosen candidates' errors (B, k) under the routing weights, plus `score_weight` times the
    divergence of the scores from softmax(-errors / temperature) over the chosen candidates (empty slots left out, whatever
    their error).  Errors get their gradient through the first term only."""
    if not temperature > 0.0:
        raise ValueError(f"temperature must be positive, got {temperature}")
    if errors.shape != routing.indices.shape:
        raise ValueError(f"errors must have shape {tuple(routing.indices.shape)}, got {tuple(errors.shape)}")
    expected = (routing.weights * torch.where(routing.indices < 0, 0.0, errors)).sum(1)  # (0 times a NaN would be NaN)
    teacher = (errors.detach() / -float(temperature)).to(torch.float32)
    return expected + score_weight * distill_top_logits(scores, teacher, routing.indices, reduction="none")
