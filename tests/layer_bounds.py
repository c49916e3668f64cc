"""Plain dense layers and norms in 64 bits, and how far a kernel's outputs may be from them.

Every bound follows the arithmetic: a rounding to type t is off by at most eps(t)/2 of the value (half a step), the
tensor cores truncate each of their sums (one step, 2^-23 of the magnitudes summed so far), float32 operations round to
half a step (2^-24).  Sums are bounded by the sum of magnitudes of their terms."""
import math

import torch

D = torch.float64
STEP = 2.0**-23          # one float32 step, relative
TINY = 2.0**-126         # below the smallest normal float32 nothing is promised


def half(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half a step of the type's subnormals."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def activation(z, name, omega):
    """act, act', and bounds of |act'| and |act''|."""
    one = torch.ones_like(z)
    if name == "relu":
        return z.clamp_min(0), (z > 0).to(D), 1.0, 0.0
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p)), 1.1, 0.5
    if name == "gelu":
        c = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 1.13, 0.8
    if name == "sin":
        return torch.sin(omega * z), omega * torch.cos(omega * z), abs(omega), omega * omega
    return z, one, 1.0, 0.0


def sum_steps(k, dtype):
    """Steps by which a sum of k products may be off, relative to the magnitudes: 16-bit products are exact and are
    accumulated 16 (or, 8 bits, 32) at a time; float32 ones lose 2 steps to what is left out of them and are accumulated
    over 512 before a rounded addition of two sums each.  Where there are few tiles the sums are split into parts of 256
    products or more, whose additions are rounded too."""
    if dtype == torch.float32:
        return min(math.ceil(k / 16), 32) + math.ceil(k / 512) + math.ceil(k / 256) + 4
    return math.ceil(k / 16) + math.ceil(k / 256) + 4


def linear(x, w, b, name, r, omega):
    """y, z, act'(z) and the bound of z's error, of 2-D operands of one type."""
    xd, wd = x.to(D), w.to(D)
    z, mag = xd @ wd.T, xd.abs() @ wd.abs().T
    if b is not None:
        z, mag = z + b.to(D), mag + b.to(D).abs()
    a, d, l1, l2 = activation(z, name, omega)
    y = a if r is None else a + r.to(D)
    ez = (sum_steps(x.shape[1], x.dtype) + 1) * STEP * mag + TINY
    return y, z, a, d, ez, l1, l2


def forward_bound(y, z, a, ez, l1, name, r, omega, out):
    """What y may be off by: the sum's error through the activation, the activation's own, the residual's addition and
    the rounding.  float32 activations are good to 8 steps of their value or argument; those rounded to 16 bits afterwards
    to 2^-19."""
    own = 0.0 if name in ("none", "relu") else (8 * STEP if out == torch.float32 else 2.0**-19)
    phase = abs(omega) * z.abs() * STEP if name == "sin" else 0.0
    e = l1 * ez + own * (a.abs() + (z.abs() if name in ("silu", "gelu") else 1.0)) * (own > 0) + phase
    if r is not None:
        e = e + STEP * (a.abs() + r.to(D).abs())
    return e * (1 + half(out)) + half(out) * y.abs() + smallest(out)


def backward(x, w, b, name, r, omega, dy, out):
    """Gradients and their bounds: {"x": (value, bound), ...}.  Elements of relu within the error of zero may go either way:
    the bound takes all of dy there."""
    y, z, a, d, ez, l1, l2 = linear(x, w, b, name, r, omega)
    g = dy.to(D)
    dz = g * d
    own = 0.0 if name in ("none", "relu") else (8 * STEP if out == torch.float32 else 2.0**-19)
    phase = omega * omega * z.abs() * STEP if name == "sin" else 0.0
    ed = l2 * ez + own * (1.0 + d.abs() + z.abs()) * max(1.0, abs(omega) if name == "sin" else 1.0) * (own > 0) + phase
    ed = ed + half(out) * d.abs() + smallest(out)                      # kept in the output's type
    edz = g.abs() * ed + half(out) * dz.abs() * (1 + half(out)) + smallest(out)    # and dz too
    if name == "none":
        edz = torch.zeros_like(dz)
    if name == "relu":
        # its slopes are exact; a positive value that rounds to zero in the output's type may count as zero
        near = z.abs() <= ez + smallest(out)
        edz = torch.where(near, g.abs(), torch.zeros_like(g))
    xd, wd = x.to(D), w.to(D)
    m, n = dz.shape
    res = {}
    ax = (dz.abs() + edz)
    v = dz @ wd
    e = edz @ wd.abs() + (sum_steps(n, x.dtype) + 1) * STEP * (ax @ wd.abs())
    res["x"] = (v, e * (1 + half(out)) + half(out) * v.abs() + smallest(out))
    v = dz.T @ xd
    e = edz.T @ xd.abs() + (sum_steps(m, x.dtype) + 16) * STEP * (ax.T @ xd.abs())      # and the sums of the splits
    res["weight"] = (v, e * (1 + half(out)) + half(out) * v.abs() + smallest(out))
    v = dz.sum(0)
    e = edz.sum(0) + (2 * math.sqrt(m) + 64) * STEP * ax.sum(0)      # a thread's share, the CTA's, the CTAs
    res["bias"] = (v, e * (1 + half(out)) + half(out) * v.abs() + smallest(out))
    if r is not None:
        res["residual"] = (g, torch.zeros_like(g))
    return res


def assert_within(got, want, bound, what):
    got = got.to(D)
    off = (got - want).abs()
    bad = ~(off <= bound)
    if bad.any():
        i = int(torch.argmax(torch.where(bad, off / bound, torch.zeros_like(off)).flatten()))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} beyond their bound, worst at {i}: got "
                             f"{got.flatten()[i].item()}, want {want.flatten()[i].item()} +- {bound.flatten()[i].item()}")
