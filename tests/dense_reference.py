"""Plain 64-bit restatements of the layers of any width, and how far a result may be off.

Bounds are elementwise.  A rounding to type t is off by at most eps(t) / 2 of the value, plus half the smallest subnormal.  A sum
of K products in 32 bits, whatever its order and even with truncation at every step, is off by at most K * 2^-23 times the sum of
the products' magnitudes (each of at most K additions loses less than one unit of the last place of a partial sum that is no
larger than that); products of 16-bit values are exact in 32 bits."""
import math

import torch

C, A = math.sqrt(2.0 / math.pi), 0.044715
NONE, RELU, GELU, SILU = 0, 1, 2, 3


def act(kind, z):
    if kind == RELU:
        return z.clamp(min=0)
    if kind == GELU:
        return z * torch.sigmoid(2 * C * (z + A * z ** 3))
    if kind == SILU:
        return z * torch.sigmoid(z)
    return z


def slope(kind, z):
    if kind == RELU:
        return (z > 0).to(z.dtype)
    if kind == GELU:
        s = torch.sigmoid(2 * C * (z + A * z ** 3))
        return s + z * s * (1 - s) * 2 * C * (1 + 3 * A * z * z)
    if kind == SILU:
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    return torch.ones_like(z)


def half_step(t, v):
    """What a rounding of v to type t may lose."""
    info = torch.finfo(t)
    return info.eps / 2 * v.abs() + info.tiny * info.eps / 2


# 32-bit evaluation of the activations and their slopes: the argument of the exponential is off by at most a few units of its last
# place, |2u| 2^-22 with |2u| <= 90 where the result is not negligible, and the exponential and the quotient add a few units:
# below 90 * 2^-22 + 2^-20 < 3e-5 of the value where it is small (|z| > 5, the value itself below 1e-5 |z|), and below 2e-6 of
# max(1, |z|) elsewhere; one bound covers both.
ACT_REL, ACT_ABS = 4e-5, 2e-6


def linear(x, w, b, r, kind, t):
    """(y, z, bound of y, bound of z) in 64 bits."""
    x, w = x.double(), w.double()
    z = x @ w.T
    mag = x.abs() @ w.abs().T
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    e = (x.shape[1] + 4) * 2.0 ** -23 * mag
    y = act(kind, z)
    ey = 1.13 * e  # no activation is steeper than 1.13
    if kind in (GELU, SILU):
        ey = ey + ACT_REL * y.abs() + ACT_ABS * torch.clamp(z.abs(), min=1.0, max=8.0)
    if r is not None:
        y = y + r.double()
        ey = ey + 2.0 ** -23 * (y.abs() + r.double().abs())
    return y, z, ey + half_step(t, y.abs() + ey), e + half_step(t, z.abs() + e)


def linear_backward(x, w, dz, below_kind, below_z, skip, t):
    """(dx, dw, db, their bounds) for a given dz."""
    x, w, dz = x.double(), w.double(), dz.double()
    n = x.shape[0]
    dx, mag = dz @ w, dz.abs() @ w.abs()
    e = (w.shape[0] + 4) * 2.0 ** -23 * mag
    if below_kind != NONE:
        s = slope(below_kind, below_z.double())
        e = e * 1.13 + dx.abs() * (ACT_REL + ACT_ABS * 8 if below_kind != RELU else 0.0)
        dx = dx * s
    if skip is not None:
        dx = dx + skip.double()
        e = e + 2.0 ** -23 * (dx.abs() + skip.double().abs())
    dw, emw = dz.T @ x, (n + 4) * 2.0 ** -23 * (dz.abs().T @ x.abs())
    db, emb = dz.sum(0), (n + 4) * 2.0 ** -23 * dz.abs().sum(0)
    return dx, dw, db, e + half_step(t, dx.abs() + e), emw + 1e-40, emb + 1e-40


def layer_norm(x, gamma, beta, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    y = (x - mean) * rstd * gamma.double()
    return (y if beta is None else y + beta.double()), mean[:, 0], rstd[:, 0]


def layer_norm_backward(x, gamma, mean, rstd, dy, skip):
    x, dy, mean, rstd = x.double(), dy.double(), mean.double()[:, None], rstd.double()[:, None]
    xh, a = (x - mean) * rstd, dy * gamma.double()
    dx = rstd * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    return (dx if skip is None else dx + skip.double()), (dy * xh).sum(0), dy.sum(0)


def within(name, got, want, bound):
    off = (got.double() - want).abs()
    ok = (off <= bound) | (got.double() == want) | (torch.isnan(got.double()) & torch.isnan(want))
    if not bool(ok.all()):
        i = int((~ok).flatten().nonzero()[0])
        raise AssertionError(f"{name}: {int((~ok).sum())} of {ok.numel()} off, first at {i}: got {got.flatten()[i].item()!r}, want "
                             f"{want.flatten()[i].item()!r}, bound {bound.expand_as(want).flatten()[i].item():.3g}")
