"""route_candidates (ur_route_forward / _backward) against the definition in 64 bits.

Indices and counts: equal.  Weights: a score is a ratio of exponentials, each within 4 roundings (u = 2^-24) of its value
plus u |l - max| of its rounded argument, and a sum of at most 1024 of them in at most 16 serial steps and 6 exchanges;
with logits below 30 in magnitude that is below 120 u relative.  Gradients: products of three such factors and a sum of
at most 64 terms: 8 * 64 u of the magnitudes that enter (bar), plus half a step of the logits' type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = float("inf")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def scores64(l, kind):
    """(..., E) float64 on the CPU, -inf scores 0"""
    if kind == "sigmoid":
        return torch.sigmoid(l)
    m = l.amax(-1, keepdim=True)
    e = torch.exp(l - torch.where(m == -INF, 0.0, m))
    z = e.sum(-1, keepdim=True)
    return e / torch.where(z == 0, 1.0, z)


def choose_row(l, s, bias, k, groups, top_groups, group_score):
    """one row by plain sorting, (score descending, index ascending); NaN is the largest"""
    E = len(l)
    big = lambda v: INF if math.isnan(v) else v  # noqa: E731
    nan_first = lambda v: 0 if math.isnan(v) else 1  # noqa: E731
    c = [l[e] if bias is None else s[e] + bias[e] for e in range(E)]
    ok = [l[e] != -INF and c[e] != -INF for e in range(E)]
    order = lambda v, e: (nan_first(v), -big(v), e)  # noqa: E731
    per = E // groups
    value = []
    for g in range(groups):
        members = [e for e in range(g * per, (g + 1) * per) if ok[e]]
        by = (lambda e: s[e]) if bias is None and group_score == "top2" else (lambda e: c[e])
        best = sorted((by(e) for e in members), key=lambda v: (nan_first(v), -big(v)))
        value.append(-INF if not best else best[0] if group_score == "max" else sum(best[:2]))
    kept = sorted(range(groups), key=lambda g: order(value[g], g))[:top_groups] if groups > 1 else [0]
    left = sorted((e for e in range(E) if ok[e] and e // per in kept), key=lambda e: order(c[e], e))
    return (left + [-1] * k)[:k]


def reference(logits, k, bias=None, score="softmax", groups=1, top_groups=1, group_score="max", renormalize=True,
              scale=1.0, dw=None):
    l = logits.detach().double().cpu().reshape(-1, logits.shape[-1])
    s = scores64(l, score)
    b = None if bias is None else bias.double().cpu().tolist()
    ll, sl = l.tolist(), s.tolist()
    idx = torch.tensor([choose_row(ll[i], sl[i], b, k, groups, top_groups, group_score) for i in range(len(ll))],
                       dtype=torch.int64).reshape(-1, k)
    real, at = idx >= 0, idx.clamp(min=0)
    if renormalize:  # a ratio: from the scores' logarithms, defined also where the scores themselves are 0 in 64 bits
        log_s = torch.nn.functional.logsigmoid(l) if score == "sigmoid" else l
        x = torch.where(real, log_s.gather(1, at), -INF)
        w = torch.where(real, scores64(x, "softmax"), 0.0)
    else:
        w = torch.where(real, s.gather(1, at), 0.0)
    out = {"indices": idx, "weights": scale * w,
           "counts": torch.bincount(idx[real], minlength=l.shape[1]).to(torch.int32)}
    if dw is not None:
        d = torch.where(real, dw.double().cpu().reshape(-1, k), 0.0)
        spread = lambda v: torch.zeros_like(s).scatter_add_(1, at, torch.where(real, v, 0.0))  # noqa: E731
        comp = (1 - s).gather(1, at) if score == "sigmoid" else torch.ones_like(w)
        if renormalize:  # d w_j / d log s_i = w_j ([i = j] - w_i); the softmax's own normalisation drops out
            out["grad"] = spread(scale * comp * w * (w[:, None, :] * (d[:, :, None] - d[:, None, :])).sum(2))
            mag = spread(abs(scale) * w * (w[:, None, :] * (d.abs()[:, :, None] + d.abs()[:, None, :])).sum(2))
        elif score == "sigmoid":
            out["grad"], mag = spread(scale * d * w * comp), spread(abs(scale) * d.abs() * w)
        else:
            out["grad"] = s * (spread(scale * d) - scale * (d * w).sum(1, keepdim=True))
            mag = s * (spread(abs(scale) * d.abs()) + abs(scale) * (d.abs() * w).sum(1, keepdim=True))
        out["bar"] = 8 * 64 * U * mag
    return out


def check(got, want, rel, bar=0.0, what=""):
    got = got.detach()
    eps, low = torch.finfo(got.dtype).eps, torch.finfo(got.dtype).smallest_normal
    bar = bar + (eps / 2 + rel) * want.abs() + low * eps / 2 + 1e-37
    err = (got.double().cpu().reshape(want.shape) - want).abs()
    assert bool((err <= bar).all()), f"{what}: {float((err / bar).max()):.2f} times the bar"


def make(M, E, dtype, seed, masked=0.0, spread=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    l = spread * torch.randn(M, E, generator=g, device="cuda")
    if masked:
        l = l.masked_fill(torch.rand(M, E, generator=g, device="cuda") < masked, -INF)
    bias = 0.1 * torch.randn(E, generator=g, device="cuda")
    return l.to(TYPES[dtype]), bias, g


def check_all(logits, k, dw_seed=0, **kw):
    from unicorn_amd.routing import route_candidates
    dw = torch.randn(logits.shape[:-1] + (k,), generator=torch.Generator().manual_seed(dw_seed)).cuda()
    want = reference(logits, k, dw=dw, **kw)
    x = logits.detach().requires_grad_(True)
    r = route_candidates(x, k, **kw)
    assert r.weights.dtype is torch.float32 and r.indices.dtype is torch.int64 and r.counts.dtype is torch.int32
    assert torch.equal(r.indices.cpu().reshape(-1, k), want["indices"])
    assert torch.equal(r.counts.cpu(), want["counts"])
    check(r.weights, want["weights"], 120 * U, what="weights")
    grad = torch.autograd.grad(r.weights, x, dw)[0]
    assert grad.dtype is x.dtype and grad.shape == x.shape
    check(grad, want["grad"], 240 * U, want["bar"], "grad")
    plain = route_candidates(logits.detach(), k, **kw)
    assert all(torch.equal(a, b) for a, b in zip(plain, r))
    return r, grad


CANDS = [1, 2, 3, 5, 6, 8, 9, 15, 16, 17, 24, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 200, 256, 257, 300, 511, 512,
         513, 777, 1000, 1023, 1024]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cands", CANDS)
def test_every_number_of_candidates(cands, dtype):
    for k in sorted({1, min(2, cands), min(8, cands), min(15, cands), min(16, cands), min(32, cands), min(64, cands)}):
        logits, bias, _ = make(21, cands, dtype, cands + k, masked=0.1)
        kw = dict(score=("softmax", "sigmoid")[k % 2], bias=bias if k in (1, 8, 64, 15) else None, renormalize=k != 2,
                  scale=1.0 if k < 8 else 2.5)
        check_all(logits, k, **kw)


@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("groups,per,top_groups,k", [(8, 32, 4, 8), (8, 8, 3, 6), (2, 3, 1, 2), (4, 7, 2, 5), (64, 16, 8, 12),
                                                     (64, 1, 5, 5), (3, 341, 2, 33), (5, 2, 5, 10), (16, 33, 4, 64),
                                                     (1, 40, 1, 4), (32, 4, 31, 20), (7, 64, 1, 64)])
def test_groups(groups, per, top_groups, k, with_bias, score, group_score):
    for seed, masked, dtype in ((1, 0.0, "f32"), (2, 0.3, "bf16"), (3, 0.8, "f16")):
        logits, bias, _ = make(33, groups * per, dtype, seed, masked)
        check_all(logits, k, bias=bias if with_bias else None, score=score, groups=groups, top_groups=top_groups,
                  group_score=group_score)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 7, 8, 15, 16, 17, 31, 33, 63, 65, 127, 129, 1025])
def test_row_counts(rows):
    for E, k in ((6, 2), (64, 6), (256, 8)):
        logits, bias, _ = make(rows, E, "bf16", rows, 0.05)
        check_all(logits, k, score="sigmoid", bias=bias)


def test_many_rows():
    from unicorn_amd.routing import route_candidates
    logits, bias, _ = make(200003, 48, "bf16", 5)
    r = route_candidates(logits, 4, bias=bias, score="sigmoid")
    assert int(r.counts.sum()) == 200003 * 4
    assert torch.equal(r.counts.long(), torch.bincount(r.indices.reshape(-1), minlength=48))
    for a in (0, 99999, 199000):
        want = reference(logits[a:a + 900], 4, bias=bias, score="sigmoid")
        assert torch.equal(r.indices[a:a + 900].cpu(), want["indices"])
        check(r.weights[a:a + 900], want["weights"], 120 * U)


def test_offsets_past_32_bits():
    from unicorn_amd.routing import route_candidates
    M, E = 2100000, 1024                                  # 2^31 elements and more
    logits, _, _ = make(1000, E, "bf16", 6)
    big = logits.repeat(M // 1000, 1).requires_grad_(True)
    r = route_candidates(big, 4)
    small = logits.clone().requires_grad_(True)
    q = route_candidates(small, 4)
    assert torch.equal(r.indices.view(-1, 1000, 4)[-1], q.indices) and torch.equal(r.counts, q.counts * (M // 1000))
    dw = torch.randn(1000, 4, device="cuda")
    g = torch.autograd.grad(r.weights, big, dw.repeat(M // 1000, 1))[0]
    assert torch.equal(g.view(-1, 1000, E)[-1], torch.autograd.grad(q.weights, small, dw)[0])


@pytest.mark.parametrize("cands,k", [(6, 3), (16, 4), (64, 6), (256, 8), (300, 20), (1024, 40)])
def test_ties_go_to_the_lowest_index(cands, k):
    """logits from a handful of values (and a bias from another): most of the order is ties"""
    g = torch.Generator(device="cuda").manual_seed(cands)
    values = torch.tensor([-1.5, -0.25, 0.0, 0.75, 1.0], device="cuda")
    logits = values[torch.randint(0, 5, (60, cands), generator=g, device="cuda")]
    logits[0] = 0.0
    logits[1, ::2], logits[1, 1::2] = 0.0, -0.0            # equal zeros
    few = torch.tensor([0.0, 0.125], device="cuda")[torch.randint(0, 2, (cands,), generator=g, device="cuda")]
    for bias in (None, torch.zeros(cands, device="cuda"), few):
        for score in ("softmax", "sigmoid"):
            for kw in ({}, dict(groups=2, top_groups=1), dict(groups=2, top_groups=2, group_score="top2")):
                if k <= kw.get("top_groups", 1) * (cands // kw.get("groups", 1)):
                    check_all(logits, k, bias=bias, score=score, **kw)


@pytest.mark.parametrize("cands,k", [(16, 4), (33, 10), (64, 6), (64, 20), (100, 12), (256, 8), (256, 15), (300, 16), (512, 31),
                                     (1024, 8), (1024, 63), (1024, 64)])
def test_ordered_rows(cands, k):
    """logits in order of the index: the largest all lie with a few lanes, and little can be ruled out beforehand"""
    up = torch.linspace(-2, 2, cands, device="cuda")
    half = torch.cat([up[::2], up[1::2].flip(0)])
    steps = (up * 6).round() / 6                           # runs of equal values, in order
    spike = torch.full_like(up, -1.0)
    spike[cands // 2: cands // 2 + 3] = torch.tensor([0.5, 0.25, 0.5], device="cuda")
    logits = torch.stack([up, up.flip(0), half, steps, steps.flip(0), spike] * 5)
    _, bias, _ = make(1, cands, "f32", cands)
    for b in (None, 0.01 * bias):
        for kw in ({}, dict(groups=4, top_groups=2, group_score="top2"), dict(groups=4, top_groups=3)):
            if cands % kw.get("groups", 1) == 0 and k <= kw.get("top_groups", 1) * (cands // kw.get("groups", 1)):
                check_all(logits, k, bias=b, score="sigmoid", **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("cands,k", [(40, 6), (256, 8), (1000, 12)])
def test_scores_closer_than_float32_can_tell(cands, k, score):
    """a bias that takes the scores' differences away up to the last bits of float32: the order is that of the exact sums
    (the bias is float32, so the sums differ by its rounding, far above 64 bits' error)"""
    g = torch.Generator().manual_seed(7)
    base = torch.randn(cands, generator=g)
    logits = base.repeat(50, 1).cuda()
    bias = (1.0 - scores64(base.double(), score)).float().cuda()
    want = reference(logits, k, bias=bias, score=score)
    near = scores64(base.double(), score) + bias.double().cpu()
    assert float(near.max() - near.min()) < 2e-7 and len(set(near.tolist())) > cands // 2
    r, _ = check_all(logits, k, bias=bias, score=score)
    assert torch.equal(r.indices.cpu(), want["indices"])
    if cands % 4 == 0:
        for gs in ("max", "top2"):
            check_all(logits, 2, bias=bias, score=score, groups=4, top_groups=2, group_score=gs)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("cands,k", [(6, 4), (64, 6), (256, 8)])
def test_masked_rows(cands, k, renormalize, score):
    logits, bias, _ = make(12, cands, "f32", 8)
    logits[1] = -INF                                      # nothing left
    logits[2] = -INF
    logits[2, cands - 1] = -3.0                           # one left
    logits[3, :cands - 2] = -INF                          # two left
    logits[4] = torch.finfo(torch.float32).min            # the type's lowest value everywhere: eligible, equal
    logits[5, 1:] = torch.finfo(torch.float32).min
    bias = bias.clone()
    bias[2] = -INF                                        # ruled out by the bias
    for b in (None, bias):
        r, grad = check_all(logits, k, bias=b, score=score, renormalize=renormalize)
        assert bool((r.indices[1] == -1).all()) and bool((r.weights[1] == 0).all()) and bool((grad[1] == 0).all())
        assert r.indices[2].tolist() == [cands - 1] + [-1] * (k - 1)
        assert b is None or not bool((r.indices == 2).any())
    if renormalize and score == "softmax":
        assert r.weights[2, 0] == 1.0 and bool((grad[2] == 0).all())


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("cands,k", [(6, 2), (64, 6), (256, 8), (1000, 20)])
def test_nan_and_infinity_stay_in_their_row(cands, k, score):
    from unicorn_amd.routing import route_candidates
    for bias in (None, torch.zeros(cands, device="cuda")):
        for kw in ({}, dict(groups=2, top_groups=1, group_score="top2")):
            if k > kw.get("top_groups", 1) * (cands // kw.get("groups", 1)):
                continue
            for renormalize in (True, False):
                logits, _, _ = make(8, cands, "f32", 9)
                dw = torch.ones(8, k, device="cuda")
                run = lambda l: (lambda x: (lambda r: (r, torch.autograd.grad(r.weights, x, dw)[0]))(  # noqa: E731
                    route_candidates(x, k, bias=bias, score=score, renormalize=renormalize, **kw)))(l.clone().requires_grad_(True))
                clean, cg = run(logits)
                logits[2, cands - 2] = float("nan")
                logits[5, 1] = INF
                r, g = run(logits)
                rows = [0, 1, 3, 4, 6, 7]
                assert torch.equal(r.indices[rows], clean.indices[rows]) and torch.equal(g[rows], cg[rows])
                assert torch.equal(r.weights[rows], clean.weights[rows])
                if score == "softmax":                     # a NaN is in every score of its row
                    assert bool(torch.isnan(r.weights[2]).all()) and bool(torch.isnan(g[2]).any())
                    assert bool(torch.isnan(r.weights[5]).any())
                else:
                    assert r.indices[2, 0] == cands - 2 and bool(torch.isnan(r.weights[2, 0]))
                    assert r.indices[5, 0] == 1 and bool(torch.isfinite(r.weights[5]).all())
                assert int(r.counts.sum()) == 8 * k


def test_tiny_scores_still_share():
    """renormalised weights are ratios: they hold where the scores themselves are below the smallest float32"""
    from unicorn_amd.routing import route_candidates
    logits = torch.tensor([[-200.0, -201.0, -202.0, 0.0]], device="cuda")
    bias = torch.tensor([3.0, 2.0, 0.0, -9.0], device="cuda")
    want = torch.tensor([[1 / (1 + math.exp(-1)), math.exp(-1) / (1 + math.exp(-1))]], dtype=torch.float64)
    for score in ("softmax", "sigmoid"):
        r = route_candidates(logits, 2, bias=bias, score=score)
        assert r.indices.tolist() == [[0, 1]]
        check(r.weights, want, 300 * U)


def test_strides_shapes_and_empty_batches():
    from unicorn_amd.routing import route_candidates
    logits, bias, _ = make(24, 30, "bf16", 10)
    base = route_candidates(logits, 3, bias=bias)
    big = torch.zeros(24, 47, dtype=torch.bfloat16, device="cuda")
    big[:, 3:33] = logits
    for v in (big[:, 3:33], logits.t().contiguous().t(), logits.repeat_interleave(2, 0)[::2]):
        assert all(torch.equal(a, b) for a, b in zip(route_candidates(v, 3, bias=bias), base))
        check_all(v, 3, bias=bias)
    r = route_candidates(logits.view(4, 6, 30), 3, bias=bias)
    assert r.weights.shape == r.indices.shape == (4, 6, 3) and torch.equal(r.indices.view(24, 3), base.indices)
    r = route_candidates(logits[0], 3, bias=torch.stack([bias, bias], 1)[:, 0])
    assert r.weights.shape == (3,) and torch.equal(r.indices, base.indices[0])
    x = torch.empty(0, 30, device="cuda", requires_grad=True)
    r = route_candidates(x, 3)
    assert r.weights.shape == (0, 3) and bool((r.counts == 0).all())
    assert torch.autograd.grad(r.weights.sum(), x)[0].shape == (0, 30)
    x = logits.float().requires_grad_(True)               # an expanded upstream gradient
    r = route_candidates(x, 3, renormalize=False)
    want = reference(x, 3, renormalize=False, dw=torch.ones(24, 3))
    check(torch.autograd.grad(r.weights.sum(), x)[0], want["grad"], 240 * U, want["bar"])
    assert not r.indices.requires_grad and not r.counts.requires_grad


def test_gradient_against_differences():
    """the slope of <weights, dw> along a direction, from central differences of the 64-bit definition with the choice
    held: step 1e-5, third derivatives of order 1"""
    logits, bias, _ = make(9, 40, "f32", 11)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            r, grad = check_all(logits, 5, bias=bias, score=score, renormalize=renormalize, dw_seed=3)
            dw = torch.randn((9, 5), generator=torch.Generator().manual_seed(3)).double()
            v = torch.randn(9, 40, generator=torch.Generator().manual_seed(4), dtype=torch.float64)

            def f(s):
                a = scores64(logits.double().cpu() + s * v, score).gather(1, r.indices.cpu())
                return float(((a / a.sum(1, keepdim=True) if renormalize else a) * dw).sum())
            slope = (f(1e-5) - f(-1e-5)) / 2e-5
            parts = grad.double().cpu() * v
            assert abs(float(parts.sum()) - slope) <= 1e-5 * float(parts.abs().sum())


def test_two_backwards_changed_inputs_streams_and_repeats():
    from unicorn_amd.routing import route_candidates
    logits, bias, _ = make(5000, 256, "bf16", 12)
    kw = dict(bias=bias, score="sigmoid", groups=8, top_groups=4, group_score="top2")
    x = logits.clone().requires_grad_(True)
    dw = torch.randn(5000, 8, device="cuda")
    r = route_candidates(x, 8, **kw)
    g = torch.autograd.grad(r.weights, x, dw, retain_graph=True)[0]
    assert torch.equal(g, torch.autograd.grad(r.weights, x, dw)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q = route_candidates(logits, 8, **kw)
    p = route_candidates(logits, 8, **kw)
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(r, q, p):
        assert torch.equal(a, b) and torch.equal(a, c)
    y = x * 1.0
    r = route_candidates(y, 8, **kw)
    y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.weights.sum().backward()
    r = route_candidates(x, 8, **kw)
    r.weights.data.mul_(1.0)                              # (.data: not counted as a change)
    torch.autograd.grad(r.weights, x, dw)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(r.weights, x, dw)
    g2 = torch.autograd.grad(route_candidates(x, 8, **kw).weights, x, dw, create_graph=True)[0]
    assert torch.equal(g2.detach(), g)
    with pytest.raises(RuntimeError, match="twice"):
        g2.float().sum().backward()


@pytest.mark.parametrize("rows,cands,k", [(32, 6, 2), (600, 256, 8)])
def test_captured_step(rows, cands, k):
    from unicorn_amd.routing import route_candidates
    logits, bias, _ = make(rows, cands, "f32", 13)
    x, dw = logits.clone().requires_grad_(True), torch.randn(rows, k, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(route_candidates(x, k, bias=bias).weights, x, dw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = route_candidates(x, k, bias=bias)
        grad = torch.autograd.grad(r.weights, x, dw)[0]
    for seed in range(4):
        l2, b2, _ = make(rows, cands, "f32", 30 + seed)
        with torch.no_grad():
            x.copy_(l2), bias.copy_(b2)
        graph.replay()
        y = l2.clone().requires_grad_(True)
        e = route_candidates(y, k, bias=b2)
        eg = torch.autograd.grad(e.weights, y, dw)[0]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(r, e)) and torch.equal(grad, eg)


def test_balance_bias_evens_out_the_choices():
    from unicorn_amd.routing import route_candidates, update_balance_bias
    logits, _, _ = make(4096, 16, "f32", 14)
    logits += torch.linspace(-1, 1, 16, device="cuda")
    bias = torch.zeros(16, device="cuda")
    first = route_candidates(logits, 2, bias=bias, score="sigmoid").counts.float()
    for _ in range(200):
        counts = route_candidates(logits, 2, bias=bias, score="sigmoid").counts
        before = bias.clone()
        assert update_balance_bias(bias, counts, 0.005) is bias
        assert torch.equal(bias, before + 0.005 * torch.sign(counts.float().mean() - counts))
    assert float(counts.float().std()) < 0.2 * float(first.std())


def test_lowest_numbers_as_biases_under_pairs_of_a_group():
    """two biases of the lowest number add up to less than float32 holds: still more than a group that has nothing eligible"""
    low = torch.finfo(torch.float32).min
    l = torch.randn(6, 12, generator=torch.Generator().manual_seed(1)).cuda()
    l[:, :3] = -INF
    l[3:, 9:] = -INF
    bias = torch.tensor([0.0] * 3 + [low] * 6 + [0.5 * low] * 3, device="cuda")
    for score in ("softmax", "sigmoid"):
        for k, top in ((1, 1), (3, 2), (5, 3)):
            check_all(l, k, bias=bias, score=score, groups=4, top_groups=top, group_score="top2")
    high = torch.tensor([0.1] * 3 + [-low] * 3 + [-0.75 * low] * 6, device="cuda")
    for k, top in ((1, 1), (3, 2), (5, 3)):
        check_all(l, k, bias=high, score="sigmoid", groups=4, top_groups=top, group_score="top2")


def test_more_rows_than_a_launch_holds_threads_for():
    from unicorn_amd.routing import route_candidates
    part = make(4096, 2, "f16", 5)[0]
    x = part.repeat(2 ** 29 // 4096 + 1, 1).requires_grad_(True)  # 8 lanes a row: 2^32 threads and some in the backward
    small = part.clone().requires_grad_(True)
    grads = []
    for t in (small, x):
        r = route_candidates(t, 1, renormalize=False)
        grads.append(torch.autograd.grad(r.weights, t, torch.ones((), device="cuda").expand_as(r.weights))[0])
    assert r.counts.sum().item() == len(x)
    assert bool((grads[1].view(-1, 8192) == grads[0].view(1, 8192)).all())


@pytest.mark.parametrize("cands,k,times", [(8, 3, 5000), (64, 6, 2500), (300, 5, 1100), (600, 9, 480)])
def test_many_rows_that_float32_cannot_order(cands, k, times):
    """scores of 1 - 1e-6 and closer: nearly every row is chosen in 64 bits, in workgroups that take many rows one after the
    other; the same rows over and over give the same"""
    from unicorn_amd.routing import route_candidates
    g = torch.Generator(device="cuda").manual_seed(cands)
    part = (14.0 + 3.0 * torch.randn(256, cands, generator=g, device="cuda")).half()
    bias = 1e-6 * torch.randn(cands, generator=g, device="cuda")
    kw = dict(bias=bias, score="sigmoid", groups=4, top_groups=2, group_score="max")
    check_all(part, k, **kw)
    small, large = route_candidates(part, k, **kw), route_candidates(part.repeat(times, 1), k, **kw)
    assert bool((large.indices.view(times, -1) == small.indices.view(1, -1)).all())
    assert bool((large.weights.view(times, -1) == small.weights.view(1, -1)).all())
    assert torch.equal(large.counts, small.counts * times)
