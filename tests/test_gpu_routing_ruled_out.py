"""route_candidates: a bias of -inf rules a candidate out whatever its score is, a NaN among them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("cands,k", [(6, 2), (16, 3), (64, 6), (128, 5), (256, 8), (100, 20), (600, 9)])
def test_a_bias_of_minus_infinity_rules_out_nan_scores(cands, k, groups, score, dtype):
    """row 0: NaN where the bias rules out, row 1: NaN elsewhere (with softmax every score of its row is NaN, and the lowest
    indices that are left are taken), row 2: both, row 3: scores close enough for 64 bits, with a NaN ruled out"""
    from unicorn_amd.routing import route_candidates
    g = torch.Generator().manual_seed(cands)
    logits = torch.randn(5, cands, generator=g)
    bias = 0.1 * torch.randn(cands, generator=g)
    out = [0, cands // 2]
    bias[out] = -INF
    logits[0, out[0]] = NAN
    logits[1, 1] = NAN
    logits[2, out], logits[2, 2] = NAN, NAN
    logits[3] = 0.0
    logits[3, out[1]] = NAN
    l = logits.to(dtype).cuda().requires_grad_(True)
    for group_score in ("max", "top2"):
        r = route_candidates(l, k, bias=bias.cuda(), score=score, groups=groups, group_score=group_score, top_groups=groups)
        chosen = r.indices.cpu()
        for e in out:
            assert not bool((chosen == e).any()), (e, chosen)
        assert int(r.counts[out].sum()) == 0 and bool((chosen >= 0).all())
        if score == "softmax":
            free = [e for e in range(cands) if e not in out]
            for row in (0, 1, 2, 3):
                assert chosen[row].tolist() == free[:k] and bool(torch.isnan(r.weights[row]).all())
            assert bool(torch.isfinite(r.weights[4]).all())
        else:
            assert chosen[1, 0] == 1 and chosen[2, 0] == 2
            assert bool(torch.isfinite(r.weights[[0, 3, 4]]).all())  # a NaN that is not chosen is in no weight


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_everything_ruled_out_beside_a_nan(score):
    from unicorn_amd.routing import route_candidates
    logits = torch.randn(3, 40, generator=torch.Generator().manual_seed(1)).cuda()
    logits[1, 7] = NAN
    r = route_candidates(logits, 4, bias=torch.full((40,), -INF, device="cuda"), score=score, groups=4, top_groups=2)
    assert bool((r.indices == -1).all()) and int(r.counts.sum()) == 0
    assert bool((r.weights[[0, 2]] == 0).all())
