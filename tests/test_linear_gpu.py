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
         (1000, 35, 131), (257, 520, 96), (300, 1100, 264), (2000, 128, 8), (640, 192, 256), (1, 5000, 3), (33, 24, 520)]


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


def test_no_wait_ran_out():
    import __ash

    assert __ash.layer_timeouts(DEV) == 0
