"""What the operators of the networks around the renderer refuse, checked without a GPU: their Python checks run before
anything touches a device, and the C entry points answer bad arguments with a code and a message before any launch (the
pointers below are never read)."""
import pytest
import torch

from unicorn_amd import native

FAKE = 4096  # a pointer that is not null; no call below gets as far as a launch


def refused(name, *args):
    rc = getattr(native.lib(), name)(*args)
    message = native.lib().ur_last_error().decode()
    assert rc < 0 and message, name
    return rc, message


def test_layer_norm_python_checks():
    from unicorn_amd.normalization import LayerNorm, layer_norm
    x = torch.randn(4, 8)
    with pytest.raises(ValueError, match="GPU"):
        layer_norm(x)
    with pytest.raises(ValueError, match="GPU"):
        layer_norm(x.requires_grad_(True))
    for bad in (torch.randn(4, 8).double(), torch.ones(4, 8, dtype=torch.int64)):
        with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
            layer_norm(bad)
    with pytest.raises(ValueError, match="at least 1"):
        layer_norm(torch.empty(4, 0))
    with pytest.raises(ValueError, match="at least 1"):
        layer_norm(torch.tensor(1.0))
    with pytest.raises(ValueError, match="weight must have shape"):
        layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="bias must have shape"):
        layer_norm(x, None, torch.ones(1, 8))
    with pytest.raises(ValueError, match="weight must be"):
        layer_norm(x, torch.ones(8).half())
    with pytest.raises(ValueError, match="same type"):
        layer_norm(x.half(), torch.ones(8).half(), torch.ones(8))
    for eps in (-1e-5, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            layer_norm(x, eps=eps)
    with pytest.raises(ValueError, match="dim"):
        LayerNorm(0)


def test_layer_norm_entry_point_checks():
    fwd = lambda x=FAKE, stride=8, w=None, b=None, dt=0, pdt=0, M=4, D=8, eps=1e-5, y=FAKE, mean=None, rstd=None, ws=None, n=0: (  # noqa: E731
        "ur_layer_norm_forward", x, stride, w, b, dt, pdt, M, D, eps, y, mean, rstd, ws, n, None)
    assert refused(*fwd(x=None))[0] == -1
    assert refused(*fwd(y=None))[0] == -1
    assert "dtype" in refused(*fwd(dt=3))[1]
    assert "type" in refused(*fwd(dt=1, pdt=2))[1]
    assert refused(*fwd(M=0))[0] == -1 and refused(*fwd(D=0))[0] == -1 and refused(*fwd(M=-1))[0] == -1
    assert refused(*fwd(M=1 << 31))[0] == -2 and refused(*fwd(D=1 << 31, stride=1 << 31))[0] == -2
    assert "stride" in refused(*fwd(stride=7))[1]
    assert "eps" in refused(*fwd(eps=-1.0))[1] and "eps" in refused(*fwd(eps=float("nan")))[1]
    assert "together" in refused(*fwd(mean=FAKE))[1]
    assert refused(*fwd(D=1 << 20, stride=1 << 20))[0] == -4          # long rows need a workspace
    n = native.lib().ur_layer_norm_workspace_bytes(1000, 8, 0, 1)
    bwd = lambda dy=FAKE, gs=8, x=FAKE, mean=FAKE, rstd=FAKE, gx=FAKE, gw=FAKE, gb=FAKE, ws=FAKE, n=n: (  # noqa: E731
        "ur_layer_norm_backward", dy, gs, x, 8, None, mean, rstd, 0, 0, 1000, 8, gx, gw, gb, ws, n, None)
    for k in ("dy", "x", "mean", "rstd"):
        assert refused(*bwd(**{k: None}))[0] == -1
    assert "no gradient" in refused(*bwd(gx=None, gw=None, gb=None))[1]
    assert "stride" in refused(*bwd(gs=7))[1]
    assert refused(*bwd(n=n - 1))[0] == -4 and refused(*bwd(ws=None))[0] == -4 and refused(*bwd(ws=FAKE + 8))[0] == -4
    for args in ((0, 8, 0, 0), (4, 0, 0, 0), (4, 8, 3, 0), (1 << 31, 8, 0, 1)):
        assert refused("ur_layer_norm_workspace_bytes", *args)[0] == -1


def test_layer_norm_workspace_sizes():
    size = native.lib().ur_layer_norm_workspace_bytes
    for dt in (0, 1, 2):
        assert size(5, 64, dt, 0) == 0                                 # rows that fit registers: nothing kept
        for M, D in ((1, 1), (7, 33), (100000, 64), (3, 1 << 20), (1, (1 << 31) - 1)):
            n = size(M, D, dt, 1)
            assert n >= (2 * D * 4 if M > 256 else 0) and n % 4 == 0    # rows of partial sums, where several workgroups sum
            assert size(M, D, dt, 0) <= n


def test_routing_python_checks():
    from unicorn_amd.routing import route_candidates
    l = torch.randn(4, 12)
    cases = [("GPU", (l, 2), {}), ("GPU", (l.clone().requires_grad_(True), 2), {}),
             ("float32, float16", (l.double(), 2), {}), ("float32, float16", (l.long(), 2), {}),
             ("at least 1", (torch.empty(3, 0), 1), {}), ("at least 1", (torch.tensor(1.0), 1), {}),
             ("score must", (l, 2), {"score": "relu"}), ("group_score must", (l, 2), {"group_score": "sum"}),
             ("groups must divide", (l, 2), {"groups": 5}), ("groups must divide", (l, 2), {"groups": 0}),
             ("top_groups must", (l, 2), {"groups": 3, "top_groups": 4}), ("top_groups must", (l, 2), {"top_groups": 0}),
             ("top_k must", (l, 0), {}), ("top_k must", (l, 13), {}), ("top_k must", (l, 5), {"groups": 3, "top_groups": 1}),
             ("finite", (l, 2), {"scale": float("inf")}), ("finite", (l, 2), {"scale": float("nan")}),
             ("bias must", (l, 2), {"bias": torch.zeros(11)}), ("bias must", (l, 2), {"bias": torch.zeros(12).half()}),
             ("bias must", (l, 2), {"bias": torch.zeros(1, 12)})]
    for match, args, kw in cases:
        with pytest.raises(ValueError, match=match):
            route_candidates(*args, **kw)
    for args, kw in (((torch.randn(2, 1025), 2), {}), ((torch.randn(2, 100), 65), {}),
                     ((torch.randn(2, 130), 2), {"groups": 65, "top_groups": 65})):
        with pytest.raises(NotImplementedError, match="at most"):
            route_candidates(*args, **kw)


def test_routing_entry_point_checks():
    def fwd(l=FAKE, stride=12, dt=0, M=1, E=12, k=2, score=0, G=1, tg=1, gs=0, scale=1.0, w=FAKE, i=FAKE, c=FAKE, ws=None, n=0):
        return refused("ur_route_forward", l, stride, dt, None, M, E, k, score, G, tg, gs, 1, scale, w, i, c, ws, n, None)
    for kw in ({"l": None}, {"w": None}, {"i": None}, {"c": None}, {"dt": 3}, {"M": 0}, {"E": 0}, {"k": 0}, {"k": 13},
               {"score": 2}, {"G": 5}, {"G": 0}, {"G": 3, "tg": 4}, {"tg": 0}, {"G": 3, "tg": 1, "k": 5}, {"gs": 2},
               {"scale": float("nan")}, {"scale": float("inf")}, {"stride": 11, "M": 2}):
        assert fwd(**kw)[0] == -1, kw
    for kw in ({"E": 1025, "stride": 1025}, {"E": 128, "stride": 128, "k": 65}, {"E": 130, "stride": 130, "G": 65, "tg": 65},
               {"M": 1 << 31}):
        assert fwd(**kw)[0] == -2, kw
    assert fwd(M=1000)[0] == -4 and fwd(M=1000, ws=FAKE + 4, n=1 << 30)[0] == -4

    def bwd(g=FAKE, l=FAKE, dt=0, M=1, E=12, w=FAKE, i=FAKE, k=2, score=0, scale=1.0, out=FAKE):
        return refused("ur_route_backward", g, l, 12, dt, M, E, w, i, k, score, 1, scale, out, None)
    for kw in ({"g": None}, {"l": None}, {"w": None}, {"i": None}, {"out": None}, {"dt": -1}, {"M": 0}, {"k": 13}, {"score": 5},
               {"scale": float("inf")}):
        assert bwd(**kw)[0] == -1, kw
    for args in ((0, 4), (4, 0), (1 << 31, 4), (4, 1025)):
        assert refused("ur_route_workspace_bytes", *args)[0] == -1
    assert native.lib().ur_route_workspace_bytes(1, 12) == 0


def test_distillation_python_checks():
    from unicorn_amd.distillation import distill_top_logits
    z, t, i = torch.randn(4, 12), torch.randn(4, 3), torch.zeros(4, 3, dtype=torch.int64)
    cases = [("GPU", (z, t, i), {}), ("GPU", (z.clone().requires_grad_(True), t, i), {}),
             ("logits must be float32", (z.double(), t, i), {}), ("teacher_logits must be float32", (z, t.double(), i), {}),
             ("int32 or int64", (z, t, i.float()), {}), ("int32 or int64", (z, t, i.short()), {}),
             ("at least 1", (torch.empty(4, 0), t, i), {}), ("at least 1", (torch.tensor(1.0), t, i), {}),
             ("must have shape", (z, t[:3], i), {}), ("must have shape", (z, t[:3], i[:3]), {}),
             ("must have shape", (z, t[:, :0], i[:, :0]), {}), ("must have shape", (z, t[0], i[0]), {}),
             ("must have shape", (z, t[None], i[None]), {}), ("reduction must", (z, t, i), {"reduction": "max"})]
    cases += [("temperature", (z, t, i), {"temperature": v}) for v in (0.0, -1.0, float("inf"), float("nan"), 1e-40)]
    for match, args, kw in cases:
        with pytest.raises(ValueError, match=match):
            distill_top_logits(*args, **kw)
    with pytest.raises(NotImplementedError, match="at most 1024"):
        distill_top_logits(z, torch.randn(4, 1025), torch.zeros(4, 1025, dtype=torch.int64))


def test_distillation_entry_point_checks():
    def fwd(z=FAKE, stride=12, dt=0, M=2, V=12, t=FAKE, tdt=0, i=FAKE, ib=8, k=3, T=1.0, red=0, loss=FAKE, ws=None, n=0):
        return refused("ur_distill_forward", z, stride, dt, M, V, t, tdt, i, ib, k, T, red, loss, None, ws, n, None)

    def bwd(g=FAKE, z=FAKE, stride=12, dt=0, M=2, V=12, t=FAKE, tdt=0, i=FAKE, ib=8, k=3, T=1.0, red=0, stats=FAKE, out=FAKE):
        return refused("ur_distill_backward", g, 1, z, stride, dt, M, V, t, tdt, i, ib, k, T, red, stats, out, None)
    both = ({"z": None}, {"t": None}, {"i": None}, {"dt": 3}, {"tdt": -1}, {"ib": 2}, {"M": 0}, {"V": 0}, {"k": 0},
            {"stride": 11}, {"T": 0.0}, {"T": -1.0}, {"T": float("nan")}, {"T": float("inf")}, {"T": 1e-45}, {"red": 3})
    for kw in both:
        assert fwd(**kw)[0] == -1 and bwd(**kw)[0] == -1, kw
    for kw in ({"k": 1025}, {"M": 1 << 31}, {"V": 1 << 31, "stride": 1 << 31}):
        assert fwd(**kw)[0] == -2 and bwd(**kw)[0] == -2, kw
    assert fwd(loss=None)[0] == -1 and bwd(g=None)[0] == -1 and bwd(stats=None)[0] == -1 and bwd(out=None)[0] == -1
    assert fwd(red=2)[0] == -4 and fwd(red=1, ws=FAKE, n=8)[0] == -4 and fwd(red=1, ws=FAKE + 8, n=1 << 20)[0] == -4
    for args in ((0, 4, 0, 0), (4, 0, 0, 0), (1 << 31, 4, 0, 0), (4, 4, 3, 0)):
        assert refused("ur_distill_workspace_bytes", *args)[0] == -1
