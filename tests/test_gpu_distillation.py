"""distill_top_logits (ur_distill_forward / _backward) against the definition in 64 bits.

Bars, with u = 2^-24, x = (z - max) / T, q = softmax(z / T):
  an exponential's argument passes 4 roundings, the exponential itself is within 2u: relative error u (4 |x| + 4);
  the sum adds at most V / 64 terms one after the other in a thread, each vector of terms may be rescaled once, then at
  most 64 partial results are merged: relative error D = u (V / 64 + 128 + 4 sum q |x|);
  a row's loss is T^2 sum p d, d = log p - log q formed in 64 bits from the two sums: T^2 D for the student's sum (whose
  128 has room for the teacher's, 2.2u); a share p is a float32 exponential of an argument reduced in 64 bits, 2u + 2^-26.5,
  over a 64-bit sum of such: below 5u, so T^2 5u sum p |d|; 2u |loss| for the roundings of the result, and reductions add
  rounded rows in 64 bits;
  a gradient is g T (q - p): |g| T (q (u (4 |x| + 8) + D) + 8u p), plus half a step of the logits' type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = float("inf")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def reference(logits, teacher, index, T=1.0, reduction="mean", g=None):
    """64 bits, on the GPU; -> dict of (value, bar)"""
    V, k = logits.shape[-1], index.shape[-1]
    z = logits.detach().double().reshape(-1, V)
    t, i = teacher.detach().double().reshape(-1, k), index.long().reshape(-1, k)
    filled = (i >= 0) & (t != -INF)
    taught = filled.any(1)
    log_p = torch.log_softmax(torch.where(filled, t / T, -INF).masked_fill(~taught[:, None], 0.0), 1)
    p = torch.where(filled, log_p.exp(), 0.0)
    at = i.clamp(min=0)
    x = (z - z.amax(1, keepdim=True)) / T
    log_q = torch.log_softmax(z / T, 1)
    q = log_q.exp()
    terms = torch.where(filled & (p > 0), p * (log_p - log_q.gather(1, at)), 0.0)
    rows = T * T * terms.sum(1)
    D = U * (V / 64 + 128 + 4 * (q * torch.where(q > 0, x.abs(), 0.0)).sum(1))
    bar = torch.where(taught, T * T * (D + 5 * U * terms.abs().sum(1)) + 2 * U * rows.abs(), 0.0)
    n = max(1, int(taught.sum()))
    if reduction == "none":
        out = {"loss": (rows, bar)}
        up = torch.ones_like(rows) if g is None else g.double().reshape(-1)
    else:
        f = 1.0 / n if reduction == "mean" else 1.0
        out = {"loss": (rows.sum() * f, bar.sum() * f)}
        up = torch.full_like(rows, f * (1.0 if g is None else float(g)))
    psum = torch.zeros_like(q).scatter_add_(1, at, p)
    up = torch.where(taught, up, 0.0)[:, None]
    ax = torch.where(q > 0, x.abs(), 0.0)
    out["grad"] = (up * T * (q - psum), up.abs() * T * (q * (U * (4 * ax + 8) + D[:, None]) + 8 * U * psum))
    out["rows"] = rows
    return out


def check(got, want, what):
    value, bar = want
    got = got.detach()
    fi = torch.finfo(got.dtype)
    bar = bar + fi.eps / 2 * value.abs() + fi.smallest_normal * fi.eps / 2 + 1e-37
    err = (got.double().reshape(value.shape) - value).abs()
    assert bool((err <= bar).all()), f"{what}: {float((err / bar).max()):.2f} times the bar"


def make(M, V, k, dtype, seed, empty=0.0, tdtype="f32", spread=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    z = spread * torch.randn(M, V, generator=gen, device="cuda")
    t = z + torch.randn(M, V, generator=gen, device="cuda")
    top = t.topk(k, 1)
    index = top.indices
    if empty:
        index = index.masked_fill(torch.rand(M, k, generator=gen, device="cuda") < empty, -1)
        index[M // 2] = -1
    return z.to(TYPES[dtype]), top.values.to(TYPES[tdtype]), index, torch.randn(M, generator=gen, device="cuda")


def run(z, t, i, T=1.0, reduction="mean", g=None):
    from unicorn_amd.distillation import distill_top_logits
    x = z.detach().requires_grad_(True)
    loss = distill_top_logits(x, t, i, temperature=T, reduction=reduction)
    return loss, torch.autograd.grad(loss, x, g)[0]


def check_all(z, t, i, T=1.0, reduction="mean", g=None):
    from unicorn_amd.distillation import distill_top_logits
    g = g if reduction == "none" else torch.tensor(0.75, device="cuda")
    want = reference(z, t, i, T, reduction, g)
    loss, grad = run(z, t, i, T, reduction, g if g.dim() == 0 else g.reshape(z.shape[:-1]))
    assert loss.dtype is torch.float32 and loss.shape == (z.shape[:-1] if reduction == "none" else ())
    assert grad.dtype is z.dtype and grad.shape == z.shape
    check(loss, want["loss"], "loss")
    check(grad, want["grad"], "grad")
    assert torch.equal(distill_top_logits(z, t, i, temperature=T, reduction=reduction), loss)
    return loss, grad


COLS = [1, 2, 3, 6, 7, 8, 9, 31, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 511, 512, 513, 642, 1000, 1023, 1024, 1025,
        1926, 2047, 2049, 4096, 4097, 8101, 16384, 16385, 32767, 32768, 32769, 65537, 131071]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cols", COLS)
def test_every_number_of_classes(cols, dtype):
    for n, k in enumerate(sorted({1, min(2, cols), min(33, cols), min(100, cols)})):
        z, t, i, g = make(9, cols, k, dtype, cols + k, empty=0.2, tdtype=("f32", dtype)[n % 2])
        check_all(z, t, i, (1.0, 2.0, 0.5, 4.0)[n], ("mean", "none", "sum", "none")[n], g)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 15, 16, 17, 63, 64, 65, 255, 257, 1000, 1025, 4100])
@pytest.mark.parametrize("cols,k,dtype", [(6, 2, "f32"), (130, 20, "bf16"), (1926, 8, "f16")])
def test_row_counts(rows, cols, k, dtype):
    z, t, i, g = make(rows, cols, k, dtype, rows, empty=0.1 if rows > 2 else 0.0)
    for reduction in ("none", "mean"):
        check_all(z, t, i, 1.5, reduction, g)


@pytest.mark.parametrize("rows,cols", [(1, 300000), (2, 1 << 20), (7, 200001), (300, 70000)])
def test_few_long_rows(rows, cols):
    for dtype in ("f32", "bf16"):
        z, t, i, g = make(rows, cols, 100, dtype, cols)
        check_all(z, t, i, 1.0, "none", g)
        check_all(z, t, i, 1.0, "mean")


def test_largest_number_of_slots():
    z, t, i, g = make(5, 5000, 1024, "bf16", 1, empty=0.1)
    check_all(z, t, i, 2.0, "none", g)
    z, t, i, g = make(5, 1024, 1024, "f32", 2)             # every class is a slot
    check_all(z, t, i, 1.0, "mean")


def test_offsets_past_32_bits():
    M, V = 16400, 131072                                   # 2^31 elements and more
    z, t, i, g = make(100, V, 8, "bf16", 3)
    want = reference(z, t, i, 1.0, "none", g)
    loss, grad = run(z.repeat(M // 100, 1), t.repeat(M // 100, 1), i.repeat(M // 100, 1), 1.0, "none", g.repeat(M // 100))
    check(loss[-100:], want["loss"], "loss")
    check(grad[-100:], want["grad"], "grad")


@pytest.mark.parametrize("cols", [6, 200, 3000, 150000])
def test_the_same_class_in_several_slots(cols):
    gen = torch.Generator(device="cuda").manual_seed(4)
    z = torch.randn(8, cols, generator=gen, device="cuda")
    t = torch.randn(8, 40, generator=gen, device="cuda")
    i = torch.randint(-2, min(cols, 5), (8, 40), generator=gen, device="cuda")   # few classes, some slots empty
    first = check_all(z, t, i, 1.0, "none", torch.ones(8, device="cuda"))
    for _ in range(3):
        again = run(z, t, i, 1.0, "none", torch.ones(8, device="cuda"))
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    i[:] = 3
    check_all(z, t, i, 1.0, "none", torch.ones(8, device="cuda"))


@pytest.mark.parametrize("cols", [6, 200, 3000, 150000])
def test_rows_without_a_teacher(cols):
    from unicorn_amd.distillation import distill_top_logits
    z, t, i, g = make(6, cols, 4, "f32", 5)
    i[1] = -1
    t[2] = -INF                                            # slots, but nothing in them
    t[3, 1:] = -INF                                        # one slot left
    i[4, :3] = -7
    z[1, 0] = float("nan")                                 # rows without a teacher are not looked at
    z[2, cols - 1] = INF
    for reduction in ("none", "mean", "sum"):
        loss, grad = run(z, t, i, 1.0, reduction, g if reduction == "none" else None)
        ok = [0, 3, 4, 5]
        want = reference(z[ok], t[ok], i[ok], 1.0, reduction, g[ok] if reduction == "none" else None)
        check(loss[ok] if reduction == "none" else loss, want["loss"], "loss")
        check(grad[ok], want["grad"], "grad")
        assert bool((grad[[1, 2]] == 0).all())
        if reduction == "none":
            assert bool((loss[[1, 2]] == 0).all())
    i[:] = -1
    for reduction in ("mean", "sum"):
        loss, grad = run(z, t, i, 1.0, reduction)
        assert float(loss.detach()) == 0.0 and bool((grad == 0).all())
    assert float(distill_top_logits(z, t, i)) == 0.0


@pytest.mark.parametrize("cols", [6, 200, 3000, 150000])
def test_infinities_and_nan_stay_in_their_row(cols):
    z, t, i, g = make(9, cols, 3, "f32", 6)
    clean_l, clean_g = run(z, t, i, 1.0, "none", g)
    low = int(z[1].argmin())
    z[1, low] = -INF                                       # a class the student rules out, not among the teacher's
    z[2, int(i[2, 0])] = -INF                              # one that the teacher wants: infinite loss, finite gradient
    z[3] = -INF
    z[4, cols - 1] = float("nan")
    z[5, 0] = INF
    t[6, 1] = float("nan")
    i[7, 2] = cols                                         # a class that there is none of
    loss, grad = run(z, t, i, 1.0, "none", g)
    for r in (0, 8):
        assert torch.equal(loss[r], clean_l[r]) and torch.equal(grad[r], clean_g[r])
    want = reference(z[1:3], t[1:3], i[1:3], 1.0, "none", g[1:3])
    check(loss[1:2], (want["loss"][0][:1], want["loss"][1][:1]), "loss")
    assert float(loss[2].detach()) == INF
    check(grad[1:3], want["grad"], "grad")
    assert float(grad[1, low]) == 0.0
    for r in (3, 4, 5, 6, 7):
        assert bool(torch.isnan(loss[r])) and bool(torch.isnan(grad[r]).all()), r


@pytest.mark.parametrize("dtype", list(TYPES))
def test_lowest_values_of_the_type(dtype):
    z, t, i, g = make(6, 300, 5, dtype, 7)
    low = torch.finfo(TYPES[dtype]).min
    z[0, 100:] = low                                       # masked classes
    z[1] = low                                             # everything masked: uniform
    i[0] = torch.arange(5, device="cuda")
    t[2, 2:] = torch.finfo(torch.float32).min
    for T in (1.0, 0.5):
        loss, grad = check_all(z, t, i, T, "none", g)
        assert bool((grad[0, 100:] == 0).all()) and bool(torch.isfinite(loss).all())


@pytest.mark.parametrize("T", [1e-3, 0.05, 1.0, 30.0, 1e4])
def test_temperatures(T):
    z, t, i, g = make(12, 700, 6, "f32", 8)
    check_all(z, t, i, T, "none", g)


def test_a_student_that_has_learnt():
    """teacher and student agree: the loss is a small difference of large logarithms"""
    z = torch.randn(10, 50, device="cuda") * 3
    i = torch.arange(50, device="cuda").repeat(10, 1)
    for noise in (0.0, 1e-3):
        t = z + noise * torch.randn_like(z)
        check_all(z, t, i, 1.0, "none", torch.ones(10, device="cuda"))


def test_layouts_and_index_types():
    z, t, i, g = make(24, 111, 5, "bf16", 9, empty=0.1)
    want = run(z, t, i, 2.0, "none", g)
    big = torch.zeros(24, 130, dtype=torch.bfloat16, device="cuda")
    big[:, 7:118] = z
    for v in (big[:, 7:118], z.t().contiguous().t(), z.repeat_interleave(2, 0)[::2]):
        assert all(torch.equal(a, b) for a, b in zip(run(v, t, i, 2.0, "none", g), want))
    for tt, ii in ((t, i.int()), (t.t().contiguous().t(), i.t().contiguous().t()), (t, i.int().repeat(1, 2)[:, :5])):
        assert all(torch.equal(a, b) for a, b in zip(run(z, tt, ii, 2.0, "none", g), want))
    l3, g3 = run(z.view(4, 6, 111), t.view(4, 6, 5), i.view(4, 6, 5), 2.0, "none", g.view(4, 6))
    assert l3.shape == (4, 6) and torch.equal(l3.view(24), want[0]) and torch.equal(g3.view(24, 111), want[1])
    lt, gt = run(z.view(4, 6, 111).transpose(0, 1), t.view(4, 6, 5).transpose(0, 1), i.view(4, 6, 5).transpose(0, 1), 2.0,
                 "none", g.view(4, 6).t())
    assert torch.equal(lt, l3.t()) and torch.equal(gt, g3.transpose(0, 1))
    l1, g1 = run(z[3], t[3], i[3], 2.0, "none", g[3])
    assert l1.shape == () and torch.equal(l1, want[0][3]) and torch.equal(g1, want[1][3])
    e = run(z, t, i, 2.0, "none", g[:1].expand(24))        # what .sum() hands back
    assert torch.equal(e[1], run(z, t, i, 2.0, "none", g[:1].repeat(24))[1])
    assert torch.equal(run(z, t, i, 2.0, "none", g.repeat_interleave(3)[::3])[1], want[1])


def test_empty_batches():
    from unicorn_amd.distillation import distill_top_logits
    z = torch.empty(0, 12, device="cuda", requires_grad=True)
    t, i = torch.empty(0, 3, device="cuda"), torch.empty(0, 3, dtype=torch.int64, device="cuda")
    for reduction in ("none", "sum", "mean"):
        loss = distill_top_logits(z, t, i, reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ()) and float(loss.detach().sum()) == 0.0
        assert torch.autograd.grad(loss.sum(), z)[0].shape == (0, 12)


def test_gradient_against_differences():
    """the slope of sum g loss along a direction, from central differences of the 64-bit definition (step 1e-5)"""
    z, t, i, g = make(7, 60, 5, "f32", 10)
    for T in (1.0, 2.0):
        loss, grad = run(z, t, i, T, "none", g)
        v = torch.randn(7, 60, device="cuda", dtype=torch.float64)
        f = lambda s: float((reference(z.double() + s * v, t, i, T, "none")["rows"] * g.double()).sum())  # noqa: E731
        slope = (f(1e-5) - f(-1e-5)) / 2e-5
        parts = grad.double() * v
        assert abs(float(parts.sum()) - slope) <= 1e-5 * float(parts.abs().sum())


def test_two_backwards_changed_inputs_streams_and_repeats():
    from unicorn_amd.distillation import distill_top_logits
    z, t, i, g = make(300, 5000, 16, "bf16", 11)
    x = z.clone().requires_grad_(True)
    loss = distill_top_logits(x, t, i)
    first = torch.autograd.grad(loss, x, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(loss, x)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(z, t, i)
    again = run(z, t, i)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other[0], loss) and torch.equal(again[0], loss)
    assert torch.equal(other[1], first) and torch.equal(again[1], first)
    y = x * 1.0
    loss = distill_top_logits(y, t, i)
    y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    loss = distill_top_logits(x, t, i)
    loss.backward(inputs=[x])
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward(inputs=[x])
    g2 = torch.autograd.grad(distill_top_logits(x, t, i), x, create_graph=True)[0]
    assert torch.equal(g2.detach(), first)
    with pytest.raises(RuntimeError, match="twice"):
        g2.float().sum().backward()
    assert not distill_top_logits(z, t.clone().requires_grad_(True), i).requires_grad   # the teacher gets none


@pytest.mark.parametrize("rows,cols,k", [(32, 6, 2), (40, 9000, 16), (2, 200000, 16)])
def test_captured_step(rows, cols, k):
    from unicorn_amd.distillation import distill_top_logits
    z, t, i, _ = make(rows, cols, k, "f32", 12)
    x = z.clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(distill_top_logits(x, t, i), x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = distill_top_logits(x, t, i)
        grad = torch.autograd.grad(loss, x)[0]
    for seed in range(4):
        z2, t2, i2, _ = make(rows, cols, k, "f32", 40 + seed, empty=0.2)
        with torch.no_grad():
            x.copy_(z2), t.copy_(t2), i.copy_(i2)
        graph.replay()
        el, eg = run(z2, t2, i2)
        torch.cuda.synchronize()
        assert torch.equal(loss, el) and torch.equal(grad, eg)


def test_more_rows_than_a_launch_holds_threads_for():
    from unicorn_amd.distillation import distill_top_logits
    g = torch.Generator(device="cuda").manual_seed(4)
    z = torch.randn(4096, 2, generator=g, device="cuda").half()
    t = torch.randn(4096, 1, generator=g, device="cuda").half()
    i = torch.randint(-1, 2, (4096, 1), generator=g, device="cuda", dtype=torch.int32)
    n = 2 ** 29 // 4096 + 1  # 8 lanes a row: 2^32 threads and some
    results = []
    for times in (1, n):
        x = z.repeat(times, 1).requires_grad_(True)
        loss = distill_top_logits(x, t.repeat(times, 1), i.repeat(times, 1), reduction="none")
        results.append((loss.detach(), torch.autograd.grad(loss, x, torch.ones((), device="cuda").expand_as(loss))[0]))
        mean = distill_top_logits(x.detach(), t.repeat(times, 1), i.repeat(times, 1))
        # the same rows over again: in 64 bits the mean differs by the roundings of 2^29 additions at most, then one to float32
        results[-1] += (mean,)
    (loss, grad, mean), (loss_n, grad_n, mean_n) = results
    assert bool((loss_n.view(-1, 4096) == loss).all()) and bool((grad_n.view(-1, 8192) == grad.view(1, 8192)).all())
    assert abs(mean_n.item() - mean.item()) <= 2 ** 29 * 2.0 ** -53 * abs(mean.item()) + 2.0 ** -24 * 2 * abs(mean.item())
