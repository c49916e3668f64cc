"""Dense layers against the formula in 64 bits, at bounds that follow their arithmetic (layer_bounds.py)."""
import pytest
import torch

import layer_bounds as lb

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "silu", "gelu", "sin"]

# rows, inputs, outputs: few rows, edges of tiles and stages, sizes that are no multiples of anything, one of everything
SIZES = [(1, 256, 256), (4, 100, 33), (3, 1, 1), (5, 64, 64), (8, 16, 16), (128, 64, 128), (129, 65, 130), (127, 8, 40),
         (1000, 35, 131), (257, 520, 96), (300, 1100, 264), (2000, 128, 8), (640, 192, 256), (1, 5000, 3), (33, 24, 520),
         # sums split over several SMs, whole and odd; more tiles than SMs with sums of several phases
         (64, 2048, 40), (65, 3001, 33), (19000, 1100, 128), (19100, 1028, 130), (150, 40, 4001)]


def make(m, k, n, dtype, seed, bias=True, residual=True, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x, w = rand(m, k).to(dtype), (rand(n, k) * scale / k**0.5).to(dtype)
    return x, w, rand(n).to(dtype) if bias else None, rand(m, n).to(dtype) if residual else None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_forward(i, dtype):
    import ash

    m, k, n = SIZES[i]
    for j, act in enumerate(ACTS):
        omega = 3.0 if act == "sin" else 1.0
        x, w, b, r = make(m, k, n, dtype, 7 * i + j, bias=(i + j) % 3 != 0, residual=(i + j) % 2 == 0)
        got = ash.fused_linear(x, w, b, activation=act, residual=r, omega=omega)
        assert got.dtype == dtype and got.shape == (m, n)
        y, z, a, d, ez, l1, l2 = lb.linear(x, w, b, act, r, omega)
        lb.assert_within(got, y, lb.forward_bound(y, z, a, ez, l1, act, r, omega, dtype), f"{act} {(m, k, n)}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_gradients(i, dtype):
    import ash

    m, k, n = SIZES[i]
    for j, act in enumerate(ACTS):
        omega = 2.0 if act == "sin" else 1.0
        x, w, b, r = make(m, k, n, dtype, 100 + 7 * i + j, bias=(i + j) % 3 != 1, residual=(i + j) % 2 == 1)
        names = [s for s, t in zip(("x", "weight", "bias", "residual"), (x, w, b, r)) if t is not None]
        leaves = [t.requires_grad_(True) for t in (x, w, b, r) if t is not None]
        y = ash.fused_linear(x, w, b, activation=act, residual=r, omega=omega)
        dy = torch.randn(m, n, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV).to(dtype)
        grads = torch.autograd.grad(y, leaves, dy)
        want = lb.backward(x.detach(), w.detach(), None if b is None else b.detach(), act,
                           None if r is None else r.detach(), omega, dy, dtype)
        for name, got in zip(names, grads):
            assert got.dtype == dtype
            lb.assert_within(got, *want[name], f"grad {name} of {act} {(m, k, n)}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5])
def test_few_outputs(n, dtype):
    """Heads: rows that are and are not whole 16-byte words, from one value on, the last group of lanes half empty, columns
    of wider rows, and both sides of the widest rows that have a kernel of their own."""
    import ash

    for i, (m, k) in enumerate(((5, 1), (33, 3), (1000, 16), (257, 64), (4099, 63), (50, 162), (301, 65), (20001, 8), (7, 64))):
        for j, act in enumerate(ACTS):
            omega = 2.0 if act == "sin" else 1.0
            x, w, b, r = make(m, k, n, dtype, 300 + 7 * i + j, bias=(i + j) % 3 != 0, residual=(i + j) % 2 == 0)
            if i % 2:      # columns of wider tables, which begin anywhere
                x, w = (torch.cat([t[:, :1], t, t[:, :j]], 1)[:, 1:1 + k] for t in (x, w))
            leaves = [t.requires_grad_(True) for t in (x, w)]
            got = ash.fused_linear(x, w, b, activation=act, residual=r, omega=omega)
            with torch.no_grad():
                y, z, a, d, ez, l1, l2 = lb.linear(x, w, b, act, r, omega)
                bound = lb.forward_bound(y, z, a, ez, l1, act, r, omega, dtype)
                for one in (got, ash.fused_linear(x, w, b, activation=act, residual=r, omega=omega)):
                    lb.assert_within(one, y, bound, f"{act} {(m, k, n)}")
            dy = make(m, 1, n, dtype, i)[3]
            want = lb.backward(x.detach(), w.detach(), b, act, r, omega, dy, dtype)
            for name, grad in zip(("x", "weight"), torch.autograd.grad(got, leaves, dy)):
                lb.assert_within(grad, *want[name], f"grad {name} of {act} {(m, k, n)}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", ["x", "weight", "bias", "residual", "x weight", "bias residual"])
def test_only_some_gradients(dtype, what):
    import ash

    for m, k, n in ((200, 63, 40), (70, 64, 64)):
        for act in ("none", "relu", "gelu"):
            x, w, b, r = make(m, k, n, dtype, 5, residual=act != "relu" or "residual" in what)
            t = {"x": x, "weight": w, "bias": b, "residual": r}
            for name in what.split():
                t[name].requires_grad_(True)
            y = ash.fused_linear(x, w, b, activation=act, residual=r)
            dy = make(m, 1, n, dtype, 6)[3]
            grads = torch.autograd.grad(y, [t[name] for name in what.split()], dy)
            d = [None if v is None else v.detach() for v in (x, w, b, r)]
            want = lb.backward(*d[:3], act, d[3], 1.0, dy, dtype)
            for name, got in zip(what.split(), grads):
                lb.assert_within(got, *want[name], f"{name} of {act}")


@pytest.mark.parametrize("dtype", TYPES)
def test_values_at_the_edges_of_the_range(dtype):
    """Zeros, the largest and the smallest values, infinities and NaN: each stays in its row."""
    import ash

    k, n = 64, 48
    x, w, b, _ = make(300, k, n, dtype, 3, residual=False)
    big = torch.finfo(dtype).max
    x[1] = 0
    x[2] = 0
    x[2, 3] = big
    x[4] = 0
    x[4, 5] = torch.finfo(dtype).smallest_normal
    x[6, 7], x[8, 9] = float("inf"), float("nan")
    w[:, 3] = torch.where(w[:, 3] < 0, -0.5, 0.5).to(dtype)
    y = ash.fused_linear(x, w, b)
    assert torch.equal(y[1], b) and bool(y[8].isnan().all()) and not bool(torch.isfinite(y[6]).any())
    rest = torch.ones(300, dtype=torch.bool, device=DEV)
    rest[[6, 8]] = False
    assert bool(torch.isfinite(y[rest]).all())
    want = (x[2, 3].double() * w[:, 3].double() + b.double())
    assert (y[2].double() - want).abs().max() <= 2 * lb.half(dtype) * big
    for act in ("relu", "silu", "gelu", "sin"):
        z = ash.fused_linear(x, w, b, activation=act)
        assert bool(z[8].isnan().all()) and bool(torch.isfinite(z[0]).all() & torch.isfinite(z[9:]).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_long_phases(dtype):
    """Sines of phases up to 2^17 by the kernel's own reduction, beyond it by the library's."""
    import ash

    x = torch.linspace(-1, 1, 4001, device=DEV)[:, None].to(dtype)
    w = torch.ones(8, 1, device=DEV, dtype=dtype)
    for omega in (1.0, 30.0, 1000.0, 1e5, 1.3e5, 1e7):
        y = ash.fused_linear(x, w, activation="sin", omega=omega)
        phase = (x.float() * omega).to(lb.D)               # the phase is a float32 product
        bound = 2.0**-20 + lb.half(dtype) if dtype != torch.float32 else 6 * lb.STEP
        assert (y.to(lb.D) - torch.sin(phase)).abs().max() <= bound, omega


def test_same_bits_again():
    import ash

    for dtype, (m, k, n) in ((torch.float32, (5000, 100, 60)), (torch.bfloat16, (65, 3001, 33)), (torch.float32, (64, 2048, 40))):
        x, w, b, r = make(m, k, n, dtype, 11)
        leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
        runs = []
        for _ in range(3):
            y = ash.fused_linear(x, w, b, "gelu", r)
            runs.append([y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))])
        assert all(torch.equal(p, q) for other in runs[1:] for p, q in zip(runs[0], other))


def test_no_wait_ran_out():
    import __ash

    assert __ash.layer_timeouts(DEV) == 0

def recorded_case(act, dtype, m, k, n, seed, scale):
    """Operands, and in 64 bits z, its error as a sum of exact products in float32, act' and act''."""
    omega = 30.0 if act == "sin" else 1.0
    x, w, b, _ = make(m, k, n, dtype, seed, residual=False, scale=scale)
    z = (x.to(lb.D) @ w.to(lb.D).T + b.to(lb.D)).requires_grad_(True)
    _, d, _, l2 = lb.activation(z, act, omega)
    d2, = torch.autograd.grad(d.sum(), z) if d.requires_grad else (torch.zeros_like(z),)
    ez = lb.linear(x.float(), w.float(), b.float(), act, None, omega)[4]
    return x, w, b, omega, z.detach(), ez, d.detach(), d2, l2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "sin"])
def test_recorded_gradients(act, dtype):
    """With create_graph the gradients keep the bounds that they have without: the slope is of the float32 sum, whatever
    the layer's type.  A sine of frequency 30 on positions, as a network's first layer has it, and layers of the usual scale."""
    import ash

    for m, k, n, scale in ((300, 3, 40, 0.58), (70, 64, 33, 1.0), (4, 64, 48, 1.0)):
        x, w, b, omega, *_ = recorded_case(act, dtype, m, k, n, 21, scale)
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        for r in (None, make(m, 1, n, dtype, 23)[3]):
            dy = make(m, 1, n, dtype, 22)[3]
            want = lb.backward(x.detach(), w.detach(), b.detach(), act, None, omega, dy, dtype)
            for create in (False, True):
                y = ash.fused_linear(x, w, b, act, r, omega)
                grads = torch.autograd.grad(y, leaves, dy, create_graph=create)
                for name, got in zip(("x", "weight", "bias"), grads):
                    lb.assert_within(got.detach(), *want[name], f"grad {name} of {act} {(m, k, n)} recorded {create}")


def test_recorded_sums_beyond_float16():
    """A float16 layer whose sums leave the type's range: the slope is that of the sum, where a rounded one would be NaN."""
    import ash

    x = torch.full((20, 64), 200.0, device=DEV, dtype=torch.float16)
    w = torch.full((8, 64), 10.0, device=DEV, dtype=torch.float16)
    w[::2] *= -1
    for act in ("silu", "gelu"):
        leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        y = ash.fused_linear(*leaves, activation=act)
        gx, = torch.autograd.grad(y, leaves[0], torch.ones_like(y), create_graph=True)
        assert torch.equal(gx, torch.full_like(gx, 40.0))      # four outputs with a slope of one, four with none


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "sin"])
def test_second_order_of_any_type(act, dtype):
    """The gradient of sum(v dx) by x and W, v constant, against the formula at bounds that follow its steps."""
    import ash

    half, own = lb.half(dtype), 32 * lb.STEP
    for m, k, n, scale in ((300, 3, 40, 0.58), (70, 64, 33, 1.0)):
        x, w, b, omega, z, ez, d, d2, l2 = recorded_case(act, dtype, m, k, n, 31, scale)
        g, v = make(m, 1, n, dtype, 32)[3], make(m, 1, k, dtype, 33)[3]
        leaves = [t.clone().requires_grad_(True) for t in (x, w)]
        y = ash.fused_linear(*leaves, b, act, omega=omega)
        gx, = torch.autograd.grad(y, leaves[0], g, create_graph=True)
        got = torch.autograd.grad((gx * v).sum(), leaves)
        x, w, g, v = (t.to(lb.D) for t in (x, w, g, v))
        scale1, scale2 = (omega, omega**2) if act == "sin" else (1.0, 1.0)
        phase = omega * z.abs() * lb.STEP if act == "sin" else 0.0
        # act' and act'' by float32 operations of terms up to 1 + z^2, of a sum off by ez; |act'''| is below 2 for these two
        e1 = l2 * ez + scale1 * (own * (1 + z.abs()) + phase)
        e2 = (omega**3 if act == "sin" else 2.0) * ez + scale2 * (own * (1 + z * z) + phase)
        dz, back = g * d, v @ w.T
        edz = g.abs() * e1 + half * dz.abs() * (1 + half) + lb.smallest(dtype)
        eback = (lb.sum_steps(k, dtype) + 1) * lb.STEP * (v.abs() @ w.abs().T)      # what comes back to dz, rounded to the type
        eback = eback * (1 + half) + half * back.abs() + lb.smallest(dtype)
        gz = g * d2 * back
        egz = g.abs() * (d2.abs() * eback + e2 * (back.abs() + eback)) + 4 * lb.STEP * gz.abs()
        final = lambda e, t: e * (1 + half) + half * t.abs() + lb.smallest(dtype)
        want = gz @ w
        e = egz @ w.abs() + (lb.sum_steps(n, torch.float32) + 1) * lb.STEP * ((gz.abs() + egz) @ w.abs())
        lb.assert_within(got[0], want, final(e, want), f"x of {act}")
        # W is reached by way of z and of the product with dz: two results of the layer's type, and their sum
        a, c = gz.T @ x, dz.T @ v
        ea = final(egz.T @ x.abs() + (lb.sum_steps(m, torch.float32) + 16) * lb.STEP * ((gz.abs() + egz).T @ x.abs()), a)
        ec = final(edz.T @ v.abs() + (lb.sum_steps(m, dtype) + 16) * lb.STEP * ((dz.abs() + edz).T @ v.abs()), c)
        lb.assert_within(got[1], a + c, final(ea + ec, a + c), f"weight of {act}")

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", [(4, 8), (2000, 8), (2000, 1), (2000, 40)])
def test_gelu_of_negative_sums(m, n, dtype):
    """The tail keeps its leading bits: value and slope relative to the terms that they are made of.  In 16 bits erfc's own
    formula is good to 2^-15 and the exponential of z^2 / 2 < 72 to 2^-15; in float32 a rounded argument costs z^2 steps."""
    import ash

    z = torch.linspace(-12, -0.5, m, device=DEV).to(dtype)[:, None].requires_grad_(True)
    y = ash.fused_linear(z, torch.ones(n, 1, device=DEV, dtype=dtype), activation="gelu")
    dz, = torch.autograd.grad(y[:, 0].sum(), z)
    again, = torch.autograd.grad(ash.fused_linear(z, torch.ones(n, 1, device=DEV, dtype=dtype), activation="gelu")[:, 0].sum(), z,
                                 create_graph=True)
    zd = z.detach().to(lb.D)
    c, d = 0.5 * torch.erfc(-zd / 2**0.5), zd * torch.exp(-zd * zd / 2) / (2 * torch.pi) ** 0.5
    rel = 2.0**-14 if dtype != torch.float32 else (16 + 4 * zd * zd) * 2.0**-24
    final = lambda e, t: e * (1 + lb.half(dtype)) + lb.half(dtype) * t.abs() + lb.smallest(dtype) + lb.TINY
    lb.assert_within(y.detach(), (zd * c).expand(m, n), final(rel * (zd * c).abs(), zd * c).expand(m, n), "gelu")
    for got in (dz, again.detach()):      # dz is rounded to the layer's type, and dx is the same value
        lb.assert_within(got, c + d, final(rel * (c.abs() + d.abs()), c + d), "its slope")

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "sin"])
def test_slopes_are_not_rounded(act, dtype):
    """One rounding of dz = dy act'(z): with rows of the unit matrix for weights dx is dz, and half a step of its type is all
    that it may be off by, beside the activation's own error.  Every way that sums leave by, and both backward passes."""
    import ash

    omega = 2.0 if act == "sin" else 1.0
    for i, (m, k, n) in enumerate(((4, 8, 8), (200, 8, 8), (3000, 8, 3), (3000, 16, 16), (3000, 33, 9), (64, 4096, 40), (50_000, 64, 64),
                                   (700, 300, 290), (2000, 1024, 512))):
        x, _, _, r = make(m, k, n, dtype, 400 + i, residual=act == "relu" and i % 2 == 0)
        dy = make(m, 1, n, dtype, 500 + i)[3]
        w = torch.eye(n, k, device=DEV, dtype=dtype)
        x.requires_grad_(True)
        dx, = torch.autograd.grad(ash.fused_linear(x, w, activation=act, residual=r, omega=omega), x, dy)
        z, g = x.detach()[:, :n].to(lb.D), dy.to(lb.D)
        _, d, _, _ = lb.activation(z, act, omega)
        assert not bool(dx[:, n:].any())
        if act == "relu":
            assert torch.equal(dx[:, :n], torch.where(x[:, :n] > 0, dy, 0))
            continue
        own = (8 * lb.STEP if dtype == torch.float32 else 2.0**-19) * (1 + d.abs() + z.abs()) * omega + omega * omega * z.abs() * lb.STEP
        e = g.abs() * own + 4 * lb.STEP * (g * d).abs()
        lb.assert_within(dx[:, :n], g * d, e * (1 + lb.half(dtype)) + lb.half(dtype) * (g * d).abs() + lb.smallest(dtype), f"{act} {(m, k, n)}")
