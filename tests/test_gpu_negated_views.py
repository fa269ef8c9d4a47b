"""Lazily negated tensors (the sign is a bit of the tensor, its memory holds the opposite numbers) as inputs and gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu

neg = torch._neg_view


def data(seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(6, 16, generator=g).cuda(), torch.randn(16, generator=g).cuda(), torch.randn(16, generator=g).cuda()


def test_layer_norm():
    from unicorn_amd.normalization import layer_norm
    x, w, b = data()
    dy = data(2)[0]
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = layer_norm(*[-t for t in leaves])
    got = layer_norm(*[neg(t) for t in leaves])
    assert neg(x).is_neg() and torch.equal(got, want)
    for a, c in zip(torch.autograd.grad(got, leaves, neg(dy)), torch.autograd.grad(want, leaves, -dy)):
        assert torch.equal(a, c)


@pytest.mark.parametrize("renormalize", [True, False])
def test_routing(renormalize):
    from unicorn_amd.routing import route_candidates
    x, bias, _ = data()
    leaf = x.clone().requires_grad_(True)
    dw = torch.randn(6, 3, generator=torch.Generator().manual_seed(3)).cuda()
    kw = dict(score="sigmoid", renormalize=renormalize)
    want = route_candidates(-leaf, 3, bias=-bias, **kw)
    got = route_candidates(neg(leaf), 3, bias=neg(bias), **kw)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    assert torch.equal(torch.autograd.grad(got.weights, leaf, neg(dw))[0], torch.autograd.grad(want.weights, leaf, -dw)[0])
    column = torch.view_as_complex(torch.randn(5, 1, 2, device="cuda")).conj().imag
    assert column.is_neg()
    weights = [route_candidates(c, 1, score="sigmoid", renormalize=False).weights for c in (column, column.clone())]
    assert torch.equal(*weights)


@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_distillation(reduction):
    from unicorn_amd.distillation import distill_top_logits
    x, _, _ = data()
    t, i = data(2)[0][:, :4].contiguous(), torch.randint(0, 16, (6, 4), generator=torch.Generator().manual_seed(4)).cuda()
    leaf = x.clone().requires_grad_(True)
    up = torch.randn((6,) if reduction == "none" else (), generator=torch.Generator().manual_seed(5)).cuda()
    want = distill_top_logits(-leaf, -t, i, reduction=reduction)
    got = distill_top_logits(neg(leaf), neg(t), neg(-i), reduction=reduction)
    assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(got, leaf, neg(up))[0], torch.autograd.grad(want, leaf, -up)[0])
