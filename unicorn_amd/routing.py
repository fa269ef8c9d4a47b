"""Routing on the HIP kernels `ur_route_forward / _backward`: which few of a row's candidates are taken, and with which
weights.  The reference predicts K candidate poses per image, renders all of them and weighs their losses by a softmax
(unicorn.py:295-304, utils/mesh.py:43-71); `Renderer.render_candidates` renders the chosen ones only.

    r = route_candidates(logits, top_k, bias=None, score="softmax", ...)      r.weights, r.indices, r.counts
    update_balance_bias(bias, r.counts, rate)                                  keeps the candidates equally often taken

The choice: scores s = softmax or sigmoid of the logits (last dimension: the candidates); c = s + bias orders them (the
bias takes part in the choice only, not in the weights, and gets no gradient); with `groups` > 1 the candidates are
consecutive groups of equal size, a group is worth its largest c ("max") or the sum of its two largest ("top2"), and only
the `top_groups` best groups take part; ties go to the lowest index.  Two scores that differ by less than float32 can
tell are still ordered as in 64 bits; without a bias the logits are compared.  (Groups whose "top2" sums agree but for the last
bit of 64 may be taken in either order.)

weights: s of the chosen, divided by their sum when `renormalize`, times `scale`; float32, largest c first, with a gradient
to the logits.  indices: int64; counts: int32, how many rows took each candidate.  A logit of -inf (or a bias of -inf) rules
a candidate out, whatever the other is; a slot that nothing is left for holds index -1 and weight 0, and adds nothing to the gradient.  NaN
counts as +inf; with "softmax" a NaN or an infinite logit makes all weights of its row NaN, with "sigmoid" a NaN that
is chosen does.
"""
from typing import NamedTuple

import torch

from . import native

MAX_CANDIDATES, MAX_CHOICES, MAX_GROUPS = 1024, 64, 64
SCORES = {"softmax": 0, "sigmoid": 1}       # UR_SCORE_*
GROUP_SCORES = {"max": 0, "top2": 1}        # UR_GROUP_*


class Routing(NamedTuple):
    weights: torch.Tensor
    indices: torch.Tensor
    counts: torch.Tensor


def route_candidates(logits, top_k, bias=None, score="softmax", groups=1, top_groups=1, group_score="max",
                     renormalize=True, scale=1.0):
    """Chooses `top_k` candidates of every row of logits (..., E).  -> Routing(weights, indices, counts)."""
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits need a last dimension of at least 1, got shape {tuple(logits.shape)}")
    native.check_type(logits, "logits")
    E = logits.shape[-1]
    if score not in SCORES:
        raise ValueError(f"score must be one of {sorted(SCORES)}, got {score!r}")
    if group_score not in GROUP_SCORES:
        raise ValueError(f"group_score must be one of {sorted(GROUP_SCORES)}, got {group_score!r}")
    if groups < 1 or E % groups:
        raise ValueError(f"groups must divide the number of candidates: {E} candidates, {groups} groups")
    if not 1 <= top_groups <= groups:
        raise ValueError(f"top_groups must be between 1 and groups = {groups}, got {top_groups}")
    if not 1 <= top_k <= top_groups * (E // groups):
        raise ValueError(f"top_k must be between 1 and the {top_groups * (E // groups)} candidates of the groups taken, "
                         f"got {top_k}")
    if E > MAX_CANDIDATES or top_k > MAX_CHOICES or groups > MAX_GROUPS:
        raise NotImplementedError(f"at most {MAX_CANDIDATES} candidates, {MAX_CHOICES} choices and {MAX_GROUPS} groups")
    scale = float(scale)
    if not abs(scale) < float("inf"):
        raise ValueError(f"scale must be finite, got {scale}")
    if bias is not None:
        if bias.shape != (E,) or bias.dtype is not torch.float32:
            raise ValueError(f"bias must be float32 of shape ({E},), got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.detach()
        bias = bias if bias.is_contiguous() else bias.contiguous()
    native.on_gpu(logits)
    return Routing(*native.nodes().route(logits, bias, top_k, SCORES[score], groups, top_groups, GROUP_SCORES[group_score],
                                         bool(renormalize), scale))


@torch.no_grad()
def update_balance_bias(bias, counts, rate):
    """In place: a candidate taken more often than the average loses `rate`, one taken less often gains it.  In a
    data-parallel job `counts` is summed over the ranks first."""
    c = counts.to(torch.float64 if counts.is_floating_point() else torch.int64)
    # against the average without dividing: float32 cannot tell counts beyond 2^24 from one another
    return bias.add_(torch.sign(torch.sub(c.sum(), c, alpha=c.numel())), alpha=float(rate))
