"""Root-mean-square norms against the formula in 64 bits, at bounds that follow their arithmetic."""
import pytest
import torch

import layer_bounds as lb

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [(1, 1), (3, 2), (7, 8), (1000, 16), (65, 33), (33, 64), (257, 65), (20, 128), (9, 1000), (5, 1024), (6, 1025),
         (3, 4096), (2, 5001), (4, 8192), (3, 8193), (2, 20000), (0, 64), (5000, 40),
         (700, 60), (1500, 9), (900, 127), (1300, 1019), (70, 1022), (40, 3230), (650, 8189), (9, 8185), (12, 7)]
EPS = 1e-6


def make(m, d, dtype, seed, residual):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)
    return ((rand(m, d) * torch.exp(rand(m, 1))).to(dtype), (1 + 0.2 * rand(d)).to(dtype),
            rand(m, d).to(dtype) if residual else None, rand(m, d).to(dtype), rand(m, d).to(dtype) if residual else None)


def exact(x, w, r, eps=EPS):
    s = x.to(lb.D) + (0 if r is None else r.to(lb.D))
    rstd = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    return s, rstd, s * rstd * w.to(lb.D)


def steps(d):
    """Float32 half steps of a row's sum: a thread's terms (32 at most, or a 256th of the row), and eight joins."""
    return max(32, d / 256) + 16


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,d", SIZES)
@pytest.mark.parametrize("residual", [False, True])
def test_norm_and_gradients(m, d, dtype, residual):
    import ash

    x, w, r, dy, ds = make(m, d, dtype, m + d, residual)
    leaves = [t.requires_grad_(True) for t in (x, w, r) if t is not None]
    got = ash.rms_norm(x, w, residual=r, eps=EPS)
    y, total = got if residual else (got, None)
    assert y.shape == (m, d) and y.dtype == dtype
    s, rstd, want = exact(x.detach(), w.detach(), None if r is None else r.detach())
    h, f = lb.half(dtype), 2.0**-24
    es = f * s.abs()                                            # one float32 addition
    rel = f * (steps(d) + 8)                                    # of rstd: half of a sum's, a root and a division
    lb.assert_within(y.detach(), want, (rel + 4 * f) * want.abs() * (1 + h) + h * want.abs() + lb.smallest(dtype), "y")
    if residual:
        lb.assert_within(total.detach(), s, es * (1 + h) + h * s.abs() + lb.smallest(dtype), "sum")
    grads = torch.autograd.grad([y] if total is None else [y, total], leaves, [dy] if ds is None else [dy, ds])
    if m == 0:
        assert all(not bool(t.any()) for t in grads)
        return
    g, wd = dy.to(lb.D), w.detach().to(lb.D)
    gw = g * wd
    c = (gw * s).mean(1, keepdim=True) * rstd**2
    dx = rstd * (gw - s * c) + (0 if ds is None else ds.to(lb.D))
    # s is read as it was rounded: half a step of its type, in s itself and in the mean
    eh = (h if residual else 0.0) + f
    mag = (gw.abs() * s.abs()).mean(1, keepdim=True) * rstd**2
    e = rstd * (gw.abs() * (rel + 4 * f) + s.abs() * mag * (2 * rel + (steps(d) + 8) * f + 2 * eh))
    e = e + f * (0 if ds is None else ds.to(lb.D).abs()) + 2 * f * dx.abs()
    bound = e * (1 + h) + h * dx.abs() + lb.smallest(dtype)
    lb.assert_within(grads[0], dx, bound, "grad x")
    if residual:
        lb.assert_within(grads[2], dx, bound, "grad residual")
    dw = (g * s * rstd).sum(0)
    most = (g * s * rstd).abs().sum(0)
    per_thread = m / 148 + 64       # rows of a thread, at least an SM's share, and the joins
    e = most * (rel + eh + f * (per_thread + 8))
    lb.assert_within(grads[1], dw, e * (1 + h) + h * dw.abs() + lb.smallest(dtype), "grad weight")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,d", SIZES)
@pytest.mark.parametrize("residual", [False, True])
def test_quantised(m, d, dtype, residual):
    import ash

    x, w, r, _, _ = make(m, d, dtype, 3 * m + d, residual)
    got = ash.rms_norm(x, w, residual=r, eps=EPS, quantize=True)
    rows, total = got if residual else (got, None)
    assert rows.codes.dtype == torch.float8_e4m3fn and rows.codes.shape == (m, d) and rows.scales.shape == (m,)
    if residual:
        assert torch.equal(total, ash.rms_norm(x, w, residual=r, eps=EPS)[1])
    if m == 0:
        return
    _, _, want = exact(x, w, r)
    rel = 2.0**-24 * (steps(d) + 16)
    scale = (want.abs().amax(1) / 448).clamp_min(2.0**-126)
    lb.assert_within(rows.scales, scale, scale * rel, "scales")
    # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below the smallest normal code; both sides of a midpoint
    back = rows.codes.to(lb.D) * rows.scales.to(lb.D)[:, None]
    lb.assert_within(back, want, want.abs() * (2.0**-4 + 4 * rel) + scale[:, None] * (2.0**-10 + 600 * rel), "values")


@pytest.mark.parametrize("d", [8, 100, 128, 4096, 9000])
def test_odd_rows(d):
    """Zeros, an infinity, a NaN and subnormals, each in a row of its own, leave the other rows alone."""
    import ash

    g = torch.Generator(device=DEV).manual_seed(d)
    x = torch.randn(6, d, generator=g, device=DEV)
    plain = ash.rms_norm(x, torch.ones(d, device=DEV))
    x[1] = 0
    x[2, d // 2] = float("inf")
    x[3, 0] = float("nan")
    x[4] *= 1e-42
    w = torch.ones(d, device=DEV)
    y, q = ash.rms_norm(x, w), ash.rms_norm(x, w, quantize=True)
    back = ash.dequantize_rows(q)
    assert torch.equal(y[[0, 5]], plain[[0, 5]])
    for t in (y, back):
        assert not bool(t[1].any()) and bool(t[3].isnan().all()) and bool(torch.isfinite(t[[0, 1, 4, 5]]).all())
    assert bool(y[2, d // 2].isnan()) and bool(back[2].isnan().all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 100])
def test_strides_offsets_and_shapes(dtype, d):
    import ash

    g = torch.Generator(device=DEV).manual_seed(1)
    wide = torch.randn(50, 3 * d + 1, generator=g, device=DEV).to(dtype)
    w = (1 + torch.randn(d + 1, generator=g, device=DEV) / 5).to(dtype)[1:]          # not aligned for wide loads
    for x in (wide[:, :d], wide[:, 1:d + 1], wide[::2, d:2 * d], wide.t()[:d].t(), wide[:1, :d].expand(50, d),
              wide[:, :d].reshape(5, 10, d)):
        r = torch.randn(x.shape, generator=g, device=DEV).to(dtype)
        got = ash.rms_norm(x, w, residual=r)
        want = ash.rms_norm(x.contiguous().clone(), w.clone(), residual=r)
        assert got[0].shape == x.shape and torch.equal(got[1], want[1])
        # rows take other paths by their alignment: sums in another order, each result within (steps + 12) half steps of
        # float32 and half a step of its type of the same value
        rtol = 2 * ((steps(d) + 12) * 2.0**-24 + lb.half(dtype))
        assert torch.allclose(got[0].float(), want[0].float(), rtol=rtol, atol=0)


def test_differences_and_second_order():
    import ash

    g = torch.Generator(device=DEV).manual_seed(5)
    x, r, dy = (torch.randn(4, 12, generator=g, device=DEV) for _ in range(3))
    w = 1 + torch.randn(12, generator=g, device=DEV) / 5
    for t in (x, w, r):
        t.requires_grad_(True)

    def first(create):
        y, s = ash.rms_norm(x, w, residual=r)
        return torch.autograd.grad([y, s], [x, w, r], [dy, dy.flip(0)], create_graph=create)

    plain, recorded = first(False), first(True)
    for a, b in zip(plain, recorded):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)      # elementwise in another order: some steps of the sum
    # the gradient of a function of the gradient, against differences of it: h^2 |f'''| / 6 and 2^-22 |f| / h, h = 2^-7
    v = torch.randn(4, 12, generator=g, device=DEV)
    second = torch.autograd.grad((recorded[0] * v).sum(), x)[0]
    h, u = 2.0**-7, torch.randn(4, 12, generator=g, device=DEV)
    ends = []
    for sign in (1, -1):
        with torch.no_grad():
            x.add_(sign * h * u)
        ends.append((first(False)[0] * v).sum().item())
        with torch.no_grad():
            x.sub_(sign * h * u)
    numeric = (ends[0] - ends[1]) / (2 * h)
    assert abs(numeric - (second * u).sum().item()) < 2e-2 * max(1.0, abs(numeric))


@pytest.mark.parametrize("made", ["same", "scaled", "normed"])
def test_second_order_with_a_residual_made_from_x(made):
    """What reaches x by way of the residual counts once, whether the backward pass is recorded or not, and the gradient of
    the recorded one is that of the formula in 64 bits."""
    import ash

    g = torch.Generator(device=DEV).manual_seed(11)
    x, dy, ds, v = (torch.randn(5, 24, generator=g, device=DEV) for _ in range(4))
    w = 1 + torch.randn(24, generator=g, device=DEV) / 5

    def formula(x, w, residual=None):
        s = x if residual is None else x + residual
        y = s * torch.rsqrt((s * s).mean(1, keepdim=True) + 1e-6) * w
        return y if residual is None else (y, s)

    def grads(norm, x, w, dy, ds, create):
        r = {"same": lambda: x, "scaled": lambda: x * 1.5, "normed": lambda: norm(x, w) * 0.5}[made]()
        return torch.autograd.grad(norm(x, w, residual=r), [x, w], [dy, ds], create_graph=create)

    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    exact = [t.detach().to(lb.D).requires_grad_(True) for t in leaves]
    want = grads(formula, *exact, dy.to(lb.D), ds.to(lb.D), True)
    for create in (False, True):
        got = grads(ash.rms_norm, *leaves, dy, ds, create)
        for a, b in zip(got, want):
            # a few dozen float32 steps of values of order ten: 2^-24 x 2^8
            assert (a.to(lb.D) - b).abs().max() <= 2.0**-16 * max(1.0, b.abs().max().item())
    second = torch.autograd.grad((got[0] * v).sum() + got[1].square().sum(), leaves)
    exact2 = torch.autograd.grad((want[0] * v.to(lb.D)).sum() + want[1].square().sum(), exact)
    for a, b in zip(second, exact2):
        # twice as many steps, of products of two such values: 2^-24 x 2^10
        assert (a.to(lb.D) - b).abs().max() <= 2.0**-14 * max(1.0, b.abs().max().item())


def test_only_the_sum_is_used():
    import ash

    x = torch.randn(5, 16, device=DEV, requires_grad=True)
    r = torch.randn(5, 16, device=DEV, requires_grad=True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    _, s = ash.rms_norm(x, w, residual=r)
    gx, gr, gw = torch.autograd.grad(s.sum(), [x, r, w], allow_unused=True)
    assert torch.equal(gx, torch.ones_like(gx)) and torch.equal(gr, gx) and gw is None
    y, _ = ash.rms_norm(x, w, residual=r)
    assert all(g is not None for g in torch.autograd.grad(y.sum(), [x, r, w]))


def test_same_bits_again():
    import ash

    x, w, r, dy, ds = make(70_001, 48, torch.float32, 9, True)
    leaves = [t.requires_grad_(True) for t in (x, w, r)]
    runs = [torch.autograd.grad(ash.rms_norm(x, w, residual=r), leaves, [dy, ds]) for _ in range(3)]
    assert all(torch.equal(a, b) for other in runs[1:] for a, b in zip(runs[0], other))

def far_rows(d, dtype, seed):
    """Rows whose squares leave the range of float32, with and without smaller values beside them."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(9, d, generator=g, device=DEV)
    big = torch.finfo(dtype).max
    x[1] *= 1e20
    x[2] = (x[2] * 1e38).clamp(-3e38, 3e38)
    x[3] = big
    x[4] *= 1e-3
    x[4, d // 2] = big
    x[6] *= 1e25
    x[7] = torch.where(x[7] > 0, x[7], -3e19)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [1, 8, 60, 100, 129, 1000, 1024, 4096, 5001, 8192, 9000])
def test_rows_whose_squares_overflow(d, dtype):
    """They have a norm like any others, in every form, and gradients."""
    import ash

    x = far_rows(d, dtype, d)
    g = torch.Generator(device=DEV).manual_seed(1)
    w = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dtype)
    dy = torch.randn(9, d, generator=g, device=DEV).to(dtype)
    s, rstd, want = exact(x, w, None)
    h, f = lb.half(dtype), 2.0**-24
    rel = f * (steps(d) + 8)
    # y is (s rstd) w: where s rstd is a float32 subnormal its rounding is half of 2^-149, times w, before y's own
    tiny = w.to(lb.D).abs() * 2.0**-150
    own = ((rel + 4 * f) * want.abs() + tiny) * (1 + h) + h * want.abs() + lb.smallest(dtype)
    lb.assert_within(ash.rms_norm(x, w), want, own, "y")
    y, total = ash.rms_norm(x, w, residual=torch.zeros_like(x))
    lb.assert_within(y, want, own, "y of a sum")
    assert torch.equal(total, x)
    rows = ash.rms_norm(x, w, quantize=True)
    scale = (want.abs().amax(1) / 448).clamp_min(2.0**-126)
    lb.assert_within(rows.scales, scale, scale * f * (steps(d) + 16), "scales")
    back = rows.codes.to(lb.D) * rows.scales.to(lb.D)[:, None]
    lb.assert_within(back, want, want.abs() * (2.0**-4 + 4 * rel) + scale[:, None] * (2.0**-10 + 600 * rel), "values")
    # the factor of a row beyond 2^126 is a subnormal number: half of its last place, 2^-150, on top
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    gd, wd = dy.to(lb.D), w.detach().to(lb.D)
    gw, n = gd * wd, s * rstd
    mean, mag = (gw * n).mean(1, keepdim=True), (gw * n).abs().mean(1, keepdim=True)
    dx = rstd * (gw - n * mean)
    er = rel + 2.0**-150 / rstd
    e = rstd * (gw.abs() * (er + 4 * f) + n.abs() * mag * (4 * er + (steps(d) + 16) * f)) + 4 * f * dx.abs() + 2.0**-148
    e = e * (1 + h) + h * dx.abs() + lb.smallest(dtype)
    dw, most = (gd * n).sum(0), ((gd * n).abs() * (er + 80 * f)).sum(0)
    for create in (False, True):
        gx, gweight = torch.autograd.grad(ash.rms_norm(x, w), leaves, dy, create_graph=create)
        lb.assert_within(gx.detach(), dx, e, f"grad x, recorded {create}")
        lb.assert_within(gweight.detach(), dw, most * (1 + h) + h * dw.abs() + lb.smallest(dtype), f"grad weight, recorded {create}")


@pytest.mark.parametrize("d", [8, 100, 129, 4096, 9000])
def test_rows_whose_squares_vanish(d):
    """Without an eps a row of tiny values has the norm of any other."""
    import ash

    g = torch.Generator(device=DEV).manual_seed(d)
    x = torch.randn(6, d, generator=g, device=DEV)
    for i, size in enumerate((1.0, 1e-15, 1e-22, 1e-30, 1e-37, 1e-42)):
        x[i] *= size
    w = 1 + 0.2 * torch.randn(d, generator=g, device=DEV)
    _, _, want = exact(x, w, None, 0.0)
    f = 2.0**-24
    own = (f * (steps(d) + 8) + 5 * f) * want.abs() + lb.smallest(torch.float32)
    lb.assert_within(ash.rms_norm(x, w, eps=0.0), want, own, "y")
    x = x[:4].clone().requires_grad_(True)      # gradients of the smaller ones leave the range
    dy = torch.randn(4, d, generator=g, device=DEV)
    s, rstd, _ = exact(x.detach(), w, None, 0.0)
    gw, n = dy.to(lb.D) * w.to(lb.D), s * rstd
    dx = rstd * (gw - n * (gw * n).mean(1, keepdim=True))
    e = rstd * (gw.abs() + n.abs() * (gw * n).abs().mean(1, keepdim=True)) * f * 8 * (steps(d) + 16)
    for create in (False, True):
        gx, = torch.autograd.grad(ash.rms_norm(x, w, eps=0.0), x, dy, create_graph=create)
        lb.assert_within(gx.detach(), dx, e, f"grad x, recorded {create}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [8, 60, 100, 129, 1000, 4096, 9000])
def test_an_infinity_or_a_nan_takes_its_row(d, dtype):
    """All of the row is NaN, in every form and in its gradient; the rows beside it are what they are without it."""
    import ash

    g = torch.Generator(device=DEV).manual_seed(d)
    x, w = torch.randn(70, d, generator=g, device=DEV).to(dtype), torch.ones(d, device=DEV, dtype=dtype)
    plain = ash.rms_norm(x, w)
    odd = torch.zeros(70, dtype=torch.bool, device=DEV)
    for row, col, value in ((3, 0, "inf"), (20, d // 2, "-inf"), (21, d - 1, "nan"), (69, d - 1, "inf")):
        x[row, col] = float(value)
        odd[row] = True
    y = ash.rms_norm(x, w)
    back = ash.dequantize_rows(ash.rms_norm(x, w, quantize=True))
    assert bool(y[odd].isnan().all()) and bool(back[odd].isnan().all()) and torch.equal(y[~odd], plain[~odd])
    assert bool(torch.isfinite(back[~odd]).all())
    x.requires_grad_(True)
    for create in (False, True):
        gx, = torch.autograd.grad(ash.rms_norm(x, w).sum(), x, create_graph=create)
        assert bool(gx[odd].isnan().all()) and bool(torch.isfinite(gx[~odd]).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_every_width_has_a_kernel(dtype):
    """Both sides of every width at which threads a row or accesses a thread change, rows whole and as columns of wider ones."""
    import ash

    edges = (1, 2, 4, 8, 16, 32, 64, 128, 256, 512, 1024, 2048, 4096, 8192)
    g = torch.Generator(device=DEV).manual_seed(2)
    h, f = lb.half(dtype), 2.0**-24
    for d in sorted({e + o for e in edges for o in (-8, -7, -4, -3, -1, 0, 1) if e + o > 0}):
        wide = torch.randn(3, d + 1, generator=g, device=DEV).to(dtype)
        w, dy = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dtype), torch.randn(3, d, generator=g, device=DEV).to(dtype)
        for x in (wide[:, :d].clone(), wide[:, 1:]):
            s, rstd, want = exact(x, w, None)
            rel = f * (steps(d) + 8)
            x = x.requires_grad_(True)
            y = ash.rms_norm(x, w)
            lb.assert_within(y.detach(), want, (rel + 4 * f) * want.abs() * (1 + h) + h * want.abs() + lb.smallest(dtype), f"y {d}")
            dx, = torch.autograd.grad(y, x, dy)
            gw, n = dy.to(lb.D) * w.to(lb.D), s * rstd
            want = rstd * (gw - n * (gw * n).mean(1, keepdim=True))
            e = rstd * (gw.abs() + n.abs() * (gw * n).abs().mean(1, keepdim=True)) * 4 * f * (steps(d) + 8)
            lb.assert_within(dx, want, e * (1 + h) + h * want.abs() + lb.smallest(dtype), f"grad {d}")
            rows = ash.rms_norm(x.detach(), w, quantize=True)
            assert torch.equal(ash.quantize_rows(y.detach()).scales.isfinite(), rows.scales.isfinite())
            back = rows.codes.to(lb.D) * rows.scales.to(lb.D)[:, None]
            scale = (s * rstd * w.to(lb.D)).abs().amax(1, keepdim=True) / 448
            lb.assert_within(back, s * rstd * w.to(lb.D), (s * rstd * w.to(lb.D)).abs() * (2.0**-4 + 4 * rel) + scale * (2.0**-10 + 600 * rel), f"codes {d}")
