"""layer_norm (ur_layer_norm_forward / _backward) against the definition in 64 bits.

Bars.  u = 2^-24 is half a step of float32, h = eps/2 of the result's type.  A row sum passes through at most 64 serial
additions in a thread (8 vectors of 8, or 16 chunk results on top of 4 vectors), 6 lane exchanges and 16 partial sums of
waves: fewer than K = 128 roundings, each of at most u times the sum of magnitudes.  So
  mean:  K u mean|x|                     (x - m) r:  K u (|h| + r mean|x|) =: K u B        (h the normalised value)
  y:     half a step of the result + 2 K u (|w| B + |b|)
  dx = r (g - c1 - h c2):   half a step + 4 K u r (|g| + mean|g| + B mean(|g| B))
  dw, db: half a step + 4 K u sum|dy| B, 4 K u sum|dy|     (fewer than 128 serial rows a thread, then 64 bits)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U, K = 2.0 ** -24, 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half(dtype):
    return 0.0 if dtype is torch.float64 else torch.finfo(dtype).eps / 2


def tiny(dtype):
    """half a step where the type's numbers are evenly spaced (subnormal results)"""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def reference(x, w, b, eps, dy=None):
    x64 = x.detach().double().reshape(-1, x.shape[-1])
    M, D = x64.shape
    w64 = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    b64 = torch.zeros(D, dtype=torch.float64, device=x.device) if b is None else b.detach().double()
    m = x64.mean(1, keepdim=True)
    r = ((x64 - m).square().mean(1, keepdim=True) + eps).rsqrt()
    h = (x64 - m) * r
    B = h.abs() + r * x64.abs().mean(1, keepdim=True)
    y = h * w64 + b64
    out = {"y": (y, 2 * K * U * (w64.abs() * B + b64.abs()))}
    if dy is not None:
        d = dy.detach().double().reshape(M, D)
        g = d * w64
        dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
        ga = g.abs()
        out["dx"] = (dx, 4 * K * U * r * (ga + ga.mean(1, keepdim=True) + B * (ga * B).mean(1, keepdim=True)))
        out["dw"] = ((d * h).sum(0), 4 * K * U * (d.abs() * B).sum(0))
        out["db"] = (d.sum(0), 4 * K * U * d.abs().sum(0))
    return out


def check(got, want, what):
    value, bar = want
    got = got.detach()
    bar = bar + half(got.dtype) * value.abs() + tiny(got.dtype)
    err = (got.double().reshape(value.shape) - value).abs()
    assert bool((err <= bar).all()), f"{what}: {float((err / bar).max()):.2f} times the bar"


def make(M, D, dtype, wtype, seed=0, affine="both"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = (rnd(M, D) * (0.3 + torch.rand(M, 1, generator=g, device="cuda")) + 2.0 * rnd(M, 1)).to(dtype)
    w = (1 + 0.3 * rnd(D)).to(wtype) if affine != "none" else None
    b = (0.3 * rnd(D)).to(wtype) if affine == "both" else None
    return x, w, b, rnd(M, D).to(dtype)


def run(x, w, b, dy, eps=1e-5):
    from unicorn_amd.normalization import layer_norm
    x = x.detach().requires_grad_(True)
    w, b = (None if p is None else p.detach().requires_grad_(True) for p in (w, b))
    y = layer_norm(x, w, b, eps)
    got = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], dy)
    out = {"y": y, "dx": got[0]}
    if w is not None:
        out["dw"] = got[1]
    if b is not None:
        out["db"] = got[-1]
    return out


def check_all(x, w, b, dy, eps=1e-5):
    from unicorn_amd.normalization import layer_norm
    want = reference(x, w, b, eps, dy)
    got = run(x, w, b, dy, eps)
    assert got["y"].dtype is x.dtype and got["y"].shape == x.shape and got["y"].is_contiguous()
    for k, v in got.items():
        check(v, want[k], k)
    assert torch.equal(layer_norm(x, w, b, eps), got["y"])  # the form without a gradient
    return got


COLS = [1, 2, 3, 7, 8, 9, 31, 63, 64, 128, 129, 255, 256, 257, 511, 512, 513, 1000, 1024, 1025, 1926, 2047, 2048, 2049,
        4096, 4097, 5000, 8191, 8192, 8193, 10240, 16384, 16385, 32768, 32769, 65536, 65537, 131072, 131080, 300001]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols", COLS)
def test_every_row_length(cols, dtype):
    rows = 1 if cols > 200000 else 5 if cols > 9000 else 37
    check_all(*make(rows, cols, TYPES[dtype], TYPES[dtype], seed=cols))


@pytest.mark.parametrize("rows", [1, 2, 3, 15, 16, 17, 63, 64, 65, 255, 1000, 4097, 20001])
@pytest.mark.parametrize("cols,dtype,wtype,affine", [(128, "f32", "f32", "both"), (642, "bf16", "f32", "weight"),
                                                     (24, "f16", "f16", "none"), (1926, "f16", "f32", "both")])
def test_row_counts(rows, cols, dtype, wtype, affine):
    check_all(*make(rows, cols, TYPES[dtype], TYPES[wtype], seed=rows, affine=affine))


def test_many_long_rows():
    """more rows than the second dimension of a grid holds (65535), each of them split over workgroups"""
    M, D = 65537, 66000
    from unicorn_amd.normalization import layer_norm
    x = torch.randn(1, D, device="cuda", dtype=torch.bfloat16).expand(M, D).contiguous()  # 8.7 GB: offsets pass 32 bits
    x[M - 1] *= 3.0
    y = layer_norm(x)
    for row in (0, 1, 32768, 65534, 65535, 65536):
        check(y[row], reference(x[row:row + 1], None, None, 1e-5)["y"], f"row {row}")
    assert torch.equal(y[0], y[65535])


def test_offsets_past_32_bits_in_the_backward():
    M, D = 65600, 32768  # 2^31 elements
    x = torch.randn(64, D, device="cuda", dtype=torch.bfloat16).repeat(M // 64, 1)
    w = torch.randn(D, device="cuda")
    got = run(x, w, None, x)
    want = reference(x[:64], w, None, 1e-5, x[:64])
    check(got["dx"][-64:], want["dx"], "dx")
    check(got["dw"], (want["dw"][0] * (M // 64), want["dw"][1] * (M // 64)), "dw")


@pytest.mark.parametrize("dtype", list(TYPES))
def test_strides_and_layouts(dtype):
    from unicorn_amd.normalization import layer_norm
    t = TYPES[dtype]
    x, w, b, dy = make(40, 77, t, t, seed=3)
    big = torch.zeros(40, 100, dtype=t, device="cuda")
    big[:, 5:82] = x                                    # rows of a wider buffer, at an odd offset
    views = {"slice": big[:, 5:82], "transposed": x.t().contiguous().t(), "every other": x.repeat_interleave(2, 0)[::2],
             "3d": x.view(5, 8, 77), "3d permuted": x.view(5, 8, 77).transpose(0, 1),
             "expanded": x[:1].expand(40, 77), "1d": x[0], "reversed copy": x.flip(0)}
    for name, v in views.items():
        assert torch.equal(layer_norm(v, w, b), layer_norm(v.contiguous(), w, b)), name
        check_all(v, w, b, dy[:v.numel() // 77].reshape(v.shape))
    g = run(x, w, b, dy)
    for gy in (dy.t().contiguous().t(), torch.cat([dy, dy], 1)[:, :77]):   # the upstream gradient's own strides
        for k, v in run(x, w, b, gy).items():
            assert torch.equal(v, g[k]), k
    s = run(x, w, b, dy[:1, :1].expand(40, 77))          # an expanded one, as .sum() makes
    for k, v in run(x, w, b, dy[:1, :1].expand(40, 77).contiguous()).items():
        assert torch.equal(v, s[k]), k
    wide = torch.stack([w, w], 1)[:, 0]                   # a strided parameter
    assert not wide.is_contiguous() and torch.equal(layer_norm(x, wide, b), layer_norm(x, w, b))


def test_rows_behind_and_beside_the_input_are_left_alone():
    from unicorn_amd import native
    x = torch.randn(9, 50, device="cuda", dtype=torch.bfloat16)
    big = torch.full((11, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    big[1:10, 3:53] = x
    before = big.clone()
    y, _ = native.nodes().layer_norm_forward(big[1:10, 3:53], None, None, 1e-5, False)
    assert torch.equal(big, before)
    check(y, reference(x, None, None, 1e-5)["y"], "y")


@pytest.mark.parametrize("dtype", list(TYPES))
def test_large_means_and_constant_rows(dtype):
    t = TYPES[dtype]
    x, w, b, dy = make(16, 500, t, torch.float32, seed=5)
    x = (x.float() + 200.0).to(t)
    x[3] = 1.5                                            # a constant row: variance 0
    x[4] = 0.0
    got = check_all(x, w, b, dy)
    assert torch.equal(got["y"][4].float(), b.to(t).float())


@pytest.mark.parametrize("cols", [5, 300, 3000, 70000])
def test_no_number_spreads_to_other_rows(cols):
    from unicorn_amd.normalization import layer_norm
    x, w, b, dy = make(6, cols, torch.float32, torch.float32, seed=6)
    clean = run(x, w, b, dy)
    bad = x.clone()
    bad[1, cols - 1], bad[3, 0], bad[4, cols // 2] = float("inf"), float("nan"), -float("inf")
    y = layer_norm(bad, w, b)
    got = run(bad, w, b, dy)
    rows = [0, 2, 5]
    assert torch.equal(y[rows], clean["y"][rows]) and torch.equal(got["dx"][rows], clean["dx"][rows])
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(got["dx"][[1, 3, 4]]).all())
    assert bool(torch.isnan(y[[1, 4]]).any(1).all())
    assert bool(torch.isnan(got["dw"]).all()) and torch.equal(got["db"], clean["db"])  # db does not read x


def test_lowest_values_of_the_type():
    for t in TYPES.values():
        x = torch.zeros(3, 64, dtype=t, device="cuda")
        x[1, ::2] = torch.finfo(t).min
        from unicorn_amd.normalization import layer_norm
        y = layer_norm(x)
        assert torch.equal(y[0], y[2]) and bool((y[0] == 0).all())
        if t is torch.float16:  # squares of 65504 fit float32: the row is normalised like any other
            check(y[1], reference(x[1:2], None, None, 1e-5)["y"], "y")


def test_empty_batches():
    from unicorn_amd.normalization import LayerNorm
    ln = LayerNorm(33, device="cuda")
    for shape in ((0, 33), (4, 0, 33)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        y = ln(x)
        assert y.shape == shape
        gx, gw, gb = torch.autograd.grad(y, (x, ln.weight, ln.bias), torch.empty_like(y))
        assert gx.shape == shape and bool((gw == 0).all()) and bool((gb == 0).all())


@pytest.mark.parametrize("cols", [96, 5000, 70000])
def test_only_the_gradients_that_are_asked_for(cols):
    from unicorn_amd.normalization import layer_norm
    x, w, b, dy = make(12, cols, torch.float32, torch.float32, seed=7)
    full = run(x, w, b, dy)
    for want_x, want_w, want_b in [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)]:
        xs, ws, bs = (t.clone().requires_grad_(bool(f)) for t, f in ((x, want_x), (w, want_w), (b, want_b)))
        layer_norm(xs, ws, bs).backward(dy)
        for t, f, k in ((xs, want_x, "dx"), (ws, want_w, "dw"), (bs, want_b, "db")):
            assert (t.grad is not None) == bool(f)
            if f:
                assert torch.equal(t.grad, full[k]), k


def test_gradient_against_differences():
    """<dx, v> + <dw, p> + <db, q> against a central difference of the 64-bit definition along (v, p, q): step 1e-4, its
    error is of the order of step^2 times the third derivative, below 1e-6 of the magnitudes here"""
    x, w, b, dy = make(7, 45, torch.float32, torch.float32, seed=8)
    got = run(x, w, b, dy)
    v, p, q = torch.randn_like(x).double(), torch.randn_like(w).double(), torch.randn_like(b).double()
    f = lambda s: float((reference(x.double() + s * v, w.double() + s * p, b.double() + s * q, 1e-5)["y"][0]  # noqa: E731
                         * dy.double()).sum())
    step = 1e-4
    slope = (f(step) - f(-step)) / (2 * step)
    parts = [(got["dx"].double() * v), (got["dw"].double() * p), (got["db"].double() * q)]
    size = sum(float(t.abs().sum()) for t in parts)
    assert abs(sum(float(t.sum()) for t in parts) - slope) <= 1e-5 * size


def test_two_backwards_and_changed_inputs():
    from unicorn_amd.normalization import layer_norm
    x, w, b, dy = make(20, 300, torch.float32, torch.float32, seed=9)
    x.requires_grad_(True)
    y = layer_norm(x, w, b)
    first = torch.autograd.grad(y, x, dy, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(y, x, dy)[0])
    z = x * 1.0
    y = layer_norm(z, w, b)
    z.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)
    y = layer_norm(x, w, b)
    torch.autograd.grad(y, x, dy)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, x, dy)
    g = torch.autograd.grad(layer_norm(x, w, b), x, dy, create_graph=True)[0]
    assert torch.equal(g.detach(), first)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()


def test_same_bits_every_time_and_on_another_stream():
    x, w, b, dy = make(3000, 642, torch.bfloat16, torch.float32, seed=10)
    first = run(x, w, b, dy)
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = run(x, w, b, dy)
        torch.cuda.current_stream().wait_stream(side)
        for k, v in run(x, w, b, dy).items():
            assert torch.equal(v, first[k]) and torch.equal(other[k], first[k]), k


@pytest.mark.parametrize("cols", [512, 70000])
def test_captured_step(cols):
    """a graph of forward and backward, replayed with new inputs between eager calls of the same sizes"""
    from unicorn_amd.normalization import layer_norm
    x, w, b, dy = make(24, cols, torch.float32, torch.float32, seed=11)
    xs, ws, bs = (t.clone().requires_grad_(True) for t in (x, w, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(layer_norm(xs, ws, bs), (xs, ws, bs), dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer_norm(xs, ws, bs)
        grads = torch.autograd.grad(y, (xs, ws, bs), dy)
    for seed in range(4):
        x2, w2, b2, dy2 = make(24, cols, torch.float32, torch.float32, seed=20 + seed)
        with torch.no_grad():
            xs.copy_(x2), ws.copy_(w2), bs.copy_(b2), dy.copy_(dy2)
        graph.replay()
        eager = run(x2, w2, b2, dy2)
        torch.cuda.synchronize()
        for k, v in zip(("y", "dx", "dw", "db"), (y,) + grads):
            assert torch.equal(v, eager[k]), k


def test_module():
    from unicorn_amd.normalization import LayerNorm, layer_norm
    x = torch.randn(6, 40, device="cuda")
    ln = LayerNorm(40, eps=1e-3, device="cuda")
    assert torch.equal(ln(x), layer_norm(x, ln.weight, ln.bias, 1e-3))
    assert [tuple(p.shape) for p in ln.parameters()] == [(40,), (40,)]
    assert list(LayerNorm(40, affine=False).parameters()) == []
    assert len(list(LayerNorm(40, bias=False).parameters())) == 1
    with pytest.raises(ValueError, match="last dimension of 40"):
        ln(torch.randn(6, 41, device="cuda"))


def test_more_rows_than_a_launch_holds_threads_for():
    from unicorn_amd.normalization import layer_norm
    part = make(4096, 2, torch.float16, torch.float16, seed=3)[0]
    x = part.repeat(2 ** 29 // 4096 + 1, 1)  # 8 lanes a row: 2^32 threads and some
    y = layer_norm(x)
    check(y[:4096], reference(part, None, None, 1e-5)["y"], "y")
    assert bool((y.view(-1, 8192) == y[:4096].view(1, 8192)).all())
