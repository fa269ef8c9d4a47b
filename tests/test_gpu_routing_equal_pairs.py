"""route_candidates where candidates are one (logit, bias) twice and others differ from them by less than float32 can tell:
saturated or tiny scores under biases that are equal or multiples of a step, as `update_balance_bias` leaves them.  Indices and
counts equal those of the 64-bit definition; weights and gradients within the bars of test_gpu_routing."""
import pytest
import torch

from test_gpu_routing import TYPES, check_all

pytestmark = pytest.mark.gpu

# every shape of a row: (candidates, choices) by lanes of a row x candidates of a lane
SHAPES = [(4, 1), (8, 3), (16, 4), (24, 5), (64, 6), (128, 8), (256, 8), (32, 20), (100, 20), (512, 20), (64, 40), (200, 40),
          (1024, 12), (1024, 64)]
# logits of which the larger ones have scores of 1 up to a few 1e-13, or of less than 1e-8
LEVELS = {"saturated": [14.0, 17.0, 20.0, 25.0, -5.0], "tiny": [-3.0, -19.0, -18.0, -20.0], "vanishing": [-150.0, -200.0, -3.0],
          "both": [-19.0, -18.0, 17.0, 20.0, 21.0, 0.5]}


def biases(E, seed):
    g = torch.Generator().manual_seed(seed)
    step = torch.zeros(E)
    for _ in range(6):                                    # six steps of 1e-3 up or down, rounded to float32 on the way
        step += 1e-3 * torch.randint(-1, 2, (E,), generator=g)
    return {"zeros": torch.zeros(E), "0.01": torch.full((E,), 0.01), "0.5": torch.full((E,), 0.5), "steps": step}


@pytest.mark.parametrize("logits,bias,k,want", [
    ([20, 20, 21], 0.0, 1, [2]), ([20, 20, 20, 30], 0.01, 1, [3]), ([3, -19, -19, -18], 0.5, 2, [0, 3]),
    ([20, 20, 25, -5], 0.0, 1, [2]), ([20] * 200 + [25], 0.0, 1, [200]), ([20] * 200 + [25, 20, 25], 0.0, 3, [200, 202, 0]),
    ([17.0] * 40 + [30.0] + [17.0] * 60, 0.01, 5, [40, 0, 1, 2, 3])])
def test_a_larger_score_behind_equal_pairs(logits, bias, k, want):
    from unicorn_amd.routing import route_candidates
    l = torch.tensor([logits, logits[::-1]], dtype=torch.float32, device="cuda")
    b = torch.full((len(logits),), bias, device="cuda")
    r = route_candidates(l, k, bias=b, score="sigmoid")
    assert r.indices[0].tolist() == want
    check_all(l, k, bias=b, score="sigmoid")


@pytest.mark.parametrize("level", list(LEVELS))
@pytest.mark.parametrize("cands,k", SHAPES)
def test_few_logits_and_equal_biases(cands, k, level):
    g = torch.Generator().manual_seed(cands + k)
    values = torch.tensor(LEVELS[level])
    logits = values[torch.randint(0, len(values), (24, cands), generator=g)]
    logits[0], logits[1] = values[0], values[1]            # all the same
    logits[2], logits[2, -1] = values[1], values[2]        # one more at the end
    logits[3], logits[3, cands // 2] = values[0], values[1]
    logits[4:8][torch.rand(4, cands, generator=g) < 0.3] = -float("inf")
    for n, (name, bias) in enumerate(biases(cands, cands).items()):
        for score in ("sigmoid", "softmax"):
            l = logits.to(TYPES[list(TYPES)[n % 3]]).cuda()
            check_all(l, k, bias=bias.cuda(), score=score)
            if n % 2 == 0 and cands % 4 == 0 and k <= cands // 2:
                for group_score in ("max", "top2"):
                    check_all(l, k, bias=bias.cuda(), score=score, groups=4, top_groups=2, group_score=group_score)


def test_many_rows_of_equal_pairs():
    """rows in several rounds of a workgroup, next to rows that are left in float32"""
    from unicorn_amd.routing import route_candidates
    g = torch.Generator().manual_seed(3)
    values = torch.tensor([14.0, 17.0, 20.0, 25.0, 0.5, -1.0])
    part = values[torch.randint(0, 6, (256, 64), generator=g)].half().cuda()
    part[::2] = torch.randn(128, 64, generator=g).half().cuda()
    bias = torch.zeros(64, device="cuda")
    check_all(part, 6, bias=bias, score="sigmoid")
    small, large = (route_candidates(p, 6, bias=bias, score="sigmoid") for p in (part, part.repeat(500, 1)))
    assert bool((large.indices.view(500, -1) == small.indices.view(1, -1)).all())
    assert torch.equal(large.counts, small.counts * 500)
