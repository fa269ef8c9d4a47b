"""The candidate step as it is used: normalise, score, choose, render the chosen, learn from their errors."""
import pytest
import torch

from unicorn_amd import synth

pytestmark = pytest.mark.gpu


def scene(B, K, level=2, seed=0):
    sc = synth.make_scene(B, level=level, tex_size=16, seed=seed, device="cuda")
    poses = synth.make_scene(B * K, level=1, tex_size=4, seed=seed + 1, device="cuda")
    from unicorn_amd.structures import Meshes, TexturesUV
    fb, ub = sc["faces"][None].expand(B, -1, -1), sc["verts_uvs"][None].expand(B, -1, -1)
    verts, maps = sc["verts"].clone().requires_grad_(True), sc["maps"].clone().requires_grad_(True)
    make = lambda v, m: Meshes(v, fb[:len(v)], TexturesUV(m, fb[:len(v)], ub[:len(v)]))  # noqa: E731
    R, T = poses["R"].view(B, K, 3, 3).clone().requires_grad_(True), poses["T"].view(B, K, 3).clone().requires_grad_(True)
    return make, verts, maps, R, T


def renderer(size=32):
    from unicorn_amd.renderer import Renderer
    return Renderer(size, cameras={"name": "fov", "fov": 30}, faces_per_pixel=8, sigma=1e-4).to("cuda")


@pytest.mark.parametrize("B,K,k", [(1, 1, 1), (3, 6, 1), (4, 6, 2), (2, 5, 5)])
def test_render_candidates_renders_the_chosen_poses(B, K, k):
    make, verts, maps, R, T = scene(B, K)
    rend = renderer()
    scores = torch.randn(B, K, device="cuda", requires_grad=True)
    bias = 0.1 * torch.randn(K, device="cuda")
    shown = rend.render_candidates(make(verts, maps), R, T, scores, k, bias=bias)
    assert shown.images.shape == (B, k, 4, 32, 32)
    key = torch.softmax(scores.detach().double(), 1) + bias.double()
    assert torch.equal(shown.routing.indices, key.sort(dim=1, descending=True, stable=True).indices[:, :k])
    for b in range(B):
        for j in range(k):
            e = int(shown.routing.indices[b, j])
            alone = rend(make(verts[b:b + 1], maps[b:b + 1]), R[b, e][None], T[b, e][None])
            assert torch.equal(shown.images[b, j], alone[0]), (b, j)
    cot = torch.randn_like(shown.images)
    loss = ((shown.images * cot).flatten(2).sum(2) * shown.routing.weights).sum()
    gR, gT, gs, gv = torch.autograd.grad(loss, (R, T, scores, verts))
    chosen = torch.zeros(B, K, dtype=torch.bool, device="cuda").scatter_(1, shown.routing.indices, True)
    assert bool((gR[~chosen] == 0).all()) and bool((gT[~chosen] == 0).all()) and bool((gs[~chosen] == 0).all())
    assert bool((gT[chosen].abs().sum(1) > 0).all()) and bool(torch.isfinite(gv).all())
    if k == 1:
        assert bool((gs == 0).all())                      # one choice has weight 1 whatever its score
    viz = rend.render_candidates(make(verts, maps), R, T, scores.detach(), k, viz_purpose=True)
    assert viz.images.shape[:3] == (B, k, 4) and torch.equal(viz.routing.counts.sum(), torch.tensor(B * k, device="cuda"))


def test_empty_slots_and_empty_batches():
    make, verts, maps, R, T = scene(3, 4)
    rend = renderer()
    scores = torch.randn(3, 4, device="cuda")
    scores[1, 1:] = -float("inf")
    scores[2] = -float("inf")
    shown = rend.render_candidates(make(verts, maps), R, T, scores, 2)
    assert shown.routing.indices[1].tolist() == [0, -1] and shown.routing.indices[2].tolist() == [-1, -1]
    assert shown.routing.weights[1].tolist() == [1.0, 0.0] and shown.routing.weights[2].tolist() == [0.0, 0.0]
    assert bool(torch.isfinite(shown.images).all())
    from unicorn_amd.candidates import candidate_loss
    x = scores.clone().requires_grad_(True)
    shown = rend.render_candidates(make(verts, maps), R, T, x, 2)
    errors = (shown.images ** 2).flatten(2).mean(2)
    loss = candidate_loss(errors, shown.routing, x, temperature=0.1)
    assert float(loss[2].detach()) == 0.0 and bool(torch.isfinite(loss[:2]).all())
    g = torch.autograd.grad(loss.sum(), x)[0]
    assert bool((g[2] == 0).all()) and bool(torch.isfinite(g).all())
    none = rend.render_candidates(make(verts[:0], maps[:0]), R[:0], T[:0], scores[:0], 2)
    assert none.images.shape == (0, 2, 4, 32, 32) and int(none.routing.counts.sum()) == 0
    viz = rend.render_candidates(make(verts[:0], maps[:0]), R[:0], T[:0], scores[:0], 2, viz_purpose=True)
    assert viz.images.shape[3:] == rend(make(verts, maps), R[:, 0], T[:, 0], viz_purpose=True).shape[2:]


def test_refusals():
    make, verts, maps, R, T = scene(2, 3)
    rend = renderer()
    scores = torch.randn(2, 3, device="cuda")
    for r, t, s in ((R[:, :2], T, scores), (R, T[:1], scores), (R, T, scores[0]), (R[:1], T[:1], scores[:1])):
        with pytest.raises(ValueError, match="render_candidates needs"):
            rend.render_candidates(make(verts, maps), r, t, s, 1)
    with pytest.raises(ValueError, match="top_k"):
        rend.render_candidates(make(verts, maps), R, T, scores, 4)


@pytest.mark.parametrize("k", [1, 2, 4])
def test_the_operators_together_against_64_bits(k):
    """latent -> layer norm -> scores -> choice -> (errors of the chosen) -> loss, with every gradient, against the same step
    in 64 bits.  Each operator is within 2^-17 of its magnitudes (their own tests); products of a few such factors and
    torch's float32 linear layer between them (64 terms) stay within 1e-4 of the largest gradient."""
    from unicorn_amd.candidates import CandidateHead, candidate_loss
    from unicorn_amd.routing import route_candidates
    torch.manual_seed(1)
    B, D, K = 24, 64, 6
    head = CandidateHead(D, K, 6).cuda()
    with torch.no_grad():
        head.norm.weight.add_(0.2 * torch.randn(D, device="cuda"))
        head.norm.bias.add_(0.2 * torch.randn(D, device="cuda"))
    z = torch.randn(B, D, device="cuda", requires_grad=True)
    bias = 0.05 * torch.randn(K, device="cuda")
    A = torch.rand(6, device="cuda")
    scores, params = head(z)
    r = route_candidates(scores, k, bias=bias)
    errors = (params * A).tanh().square().mean(2).gather(1, r.indices)
    loss = candidate_loss(errors, r, scores, temperature=0.1, score_weight=0.5)
    names = ["z", "norm.weight", "norm.bias", "score.weight", "score.bias", "params.weight", "params.bias"]
    leaves = [z] + [dict(head.named_parameters())[n] for n in names[1:]]
    got = torch.autograd.grad(loss.mean(), leaves)

    p = {n: t.detach().double().requires_grad_(True) for n, t in zip(names, leaves)}
    h = torch.nn.functional.layer_norm(p["z"], (D,), p["norm.weight"], p["norm.bias"], 1e-5)
    s64 = h @ p["score.weight"].t() + p["score.bias"]
    q = torch.softmax(s64, 1)
    idx = (q.detach() + bias.double()).sort(dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(idx, r.indices)
    w = q.gather(1, idx)
    w = w / w.sum(1, keepdim=True)
    e64 = ((h @ p["params.weight"].t() + p["params.bias"]).view(B, K, 6) * A.double()).tanh().square().mean(2).gather(1, idx)
    t = torch.softmax(-e64.detach() / 0.1, 1)
    want_loss = (w * e64).sum(1) + 0.5 * (t * (t.log() - torch.log_softmax(s64, 1).gather(1, idx))).sum(1)
    want = torch.autograd.grad(want_loss.mean(), list(p.values()))
    assert float((loss - want_loss).detach().abs().max()) <= 1e-4 * float(want_loss.detach().abs().max())
    for n, a, b in zip(names, got, want):
        assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max()), n


@pytest.mark.parametrize("top", [1, 2])
def test_training_step_with_candidates_runs(top):
    from examples.train_step import TinyUnicorn, synthetic_targets, train_steps
    torch.manual_seed(0)
    model = TinyUnicorn(32, level=2, faces_per_pixel=10, tex_size=16, latent=32, n_poses=6, top_poses=top).to("cuda")
    imgs = synthetic_targets(4, 32, seed=5, device="cuda")
    losses = train_steps(model, imgs, 6, lr=0.01)
    assert all(torch.isfinite(torch.tensor(losses)))
    assert bool((model.balance != 0).any())
    model.pose_step = True
    model.zero_grad(set_to_none=True)
    model(imgs).mean().backward()
    for name in ("norm.weight", "norm.bias", "score.weight", "params.weight"):
        g = dict(model.candidates.named_parameters())[name].grad
        assert g is not None and bool(torch.isfinite(g).all()) and float(g.abs().sum()) > 0, name
    assert model.deform.weight.grad is None and model.texture.weight.grad is None
    model.iter_step()
    model.zero_grad(set_to_none=True)
    model(imgs).mean().backward()
    assert model.candidates.params.weight.grad is None and float(model.texture.weight.grad.abs().sum()) > 0


def test_one_pose_is_what_it_was():
    """the default model has no candidate parts, and its random initialisation is not disturbed by them"""
    from examples.train_step import TinyUnicorn
    torch.manual_seed(3)
    a = TinyUnicorn(32, level=1, tex_size=8, latent=16)
    torch.manual_seed(3)
    b = TinyUnicorn(32, level=1, tex_size=8, latent=16, n_poses=6, top_poses=2)
    assert not hasattr(a, "candidates")
    for (n, p), q in zip(a.named_parameters(), b.parameters()):
        assert torch.equal(p, q), n


def test_captured_candidate_step():
    """choice and gradients of a whole step as one graph, replayed on changing latents between eager steps"""
    from unicorn_amd.candidates import CandidateHead, candidate_loss
    from unicorn_amd.routing import route_candidates
    torch.manual_seed(2)
    head = CandidateHead(128, 6, 6).cuda()
    bias, z = torch.zeros(6, device="cuda"), torch.randn(32, 128, device="cuda")
    leaves = list(head.parameters())

    def step():
        scores, params = head(z)
        r = route_candidates(scores, 2, bias=bias)
        errors = params.square().mean(2).gather(1, r.indices)
        loss = candidate_loss(errors, r, scores, temperature=0.1)
        grads = torch.autograd.grad(loss.mean(), leaves)
        return (loss.detach(), r.indices, r.counts) + grads  # (no graph of the leaves outlives the call)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        z.copy_(torch.randn(32, 128, generator=torch.Generator().manual_seed(seed)))
        bias.copy_(0.1 * torch.randn(6, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)


def _operators(x, w):
    """every operator of the step, from a leaf"""
    from unicorn_amd.distillation import distill_top_logits
    from unicorn_amd.normalization import layer_norm
    from unicorn_amd.routing import route_candidates
    index = torch.arange(2, device="cuda").repeat(len(x), 1)
    return {"layer_norm": lambda: layer_norm(x, w), "route_candidates": lambda: route_candidates(x, 2).weights,
            "distill_top_logits": lambda: distill_top_logits(x, x.detach()[:, :2].contiguous(), index)}


@pytest.mark.parametrize("name", ["layer_norm", "route_candidates", "distill_top_logits"])
def test_forward_mode_is_refused(name):
    import torch.autograd.forward_ad as fwd
    x, w = torch.randn(5, 8, device="cuda"), torch.ones(8, device="cuda")
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            _operators(dual, w)[name]()
    _operators(x, w)[name]()


@pytest.mark.parametrize("name", ["layer_norm", "route_candidates", "distill_top_logits"])
def test_captured_backward_beside_an_eager_graph_of_the_same_leaf_is_refused(name):
    """the leaf's accumulator belongs to the default stream as long as the eager graph lives; without that graph, the
    capture works"""
    x = torch.randn(5, 8, device="cuda").requires_grad_(True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    op = _operators(x, w)[name]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        op().sum().backward()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    eager = op()
    with pytest.raises(RuntimeError, match="default stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            op().sum().backward()
    eager.sum().backward()  # (the eager graph is as good as before)
    want = torch.autograd.grad(op().sum(), x)[0]
    del eager
    x.grad = w.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op().sum().backward()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x.grad, want)
