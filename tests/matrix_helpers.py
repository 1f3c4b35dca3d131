"""The matrix operators' definition in 64 bits, and an emulation of the
arithmetic the kernels document (fp16 operands, X as hi + lo, 32-bit sums),
from which the tests' tolerances are taken."""
import math

import torch

COEF = (3.4445, -4.7750, 2.0315)


def _short(x):
    return (x.transpose(-1, -2), True) if x.shape[-2] > x.shape[-1] else (x, False)


def ns64(g, steps=5, coef=COEF, eps=1e-7):
    """The definition, in 64 bits; g: [..., rows, cols]."""
    rows = [coef] * steps if not hasattr(coef[0], "__len__") else coef
    x = g.double()
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + eps)
    x, t = _short(x)
    for a, b, c in rows:
        p = x @ x.transpose(-1, -2)
        x = a * x + (b * p + c * p @ p) @ x
    return x.transpose(-1, -2) if t else x


def ns_emulated(g, three, steps=5, coef=COEF, eps=1e-7):
    """As the kernels compute it: fp16 operands, 64-bit sums (so that what is
    left is the operands' rounding alone), `three` products or one."""
    rows = [coef] * steps if not hasattr(coef[0], "__len__") else coef
    x = g.double()
    m, n = sorted(x.shape[-2:])
    sx = 2.0 ** min(12, max(6, math.floor(0.5 * math.log2(m * n))))
    x = x * (sx / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + eps))
    x, t = _short(x)

    def parts(v):
        hi = v.float().half().double()
        return hi, (v - hi).float().half().double()

    def product(p, q):
        (ph, pl), (qh, ql) = p, q
        return ph @ qh + (ph @ ql + pl @ qh if three else 0.0)

    sa = 1024.0
    for a, b, c in rows:
        xs = parts(x)
        ps = parts(product(xs, (xs[0].transpose(-1, -2), xs[1].transpose(-1, -2))) * (sa / sx / sx))
        held = ps[0] + ps[1] if three else ps[0]
        bs = parts(b * held + (c / sa) * product(ps, ps))
        x = a * (xs[0] + xs[1]) + product(bs, xs) / sa
    x = x / sx
    return x.transpose(-1, -2) if t else x


def rel(x, y):
    """2-norm of the difference over the 2-norm, over everything."""
    d = (x.double() - y.double()).norm()
    n = y.double().norm()
    return float(d / n) if float(n) else float(d)


# What 32-bit arithmetic may leave in a result of five steps, relative to it. A
# step's terms a x, b A x, c A A x are at most (3.45 + 4.78 l + 2.04 l^2) x <=
# 14.6 x for eigenvalues l <= 1.44 of A, and each is rounded at most thrice (a
# coefficient, a product, a sum), by 2^-24 of itself: 44 x 2^-24 x a step. What
# a step leaves, each later one multiplies by the slope of a s + b s^3 + c s^5,
# at most 1.71 for singular values s in [0.68, 1.13], where the iteration keeps
# them: 1 + 1.71 + ... + 1.71^4 < 19.
ARITHMETIC = 19 * 44 * 2.0 ** -24


def sums(n):
    """The tensor cores' 32-bit sums, relative to the result: a side of n takes
    n / 16 additions, each off by at most 2^-23 of the running sum, which grows
    evenly to the whole (half of it on average); a relative error of A counts
    at most |b| + 2 c < 9 times (for eigenvalues up to 1)."""
    return 9 * n / 32 * 2.0 ** -23


def tolerance(g, exact, dtype, **kw):
    """How far a result of type `dtype` may be from `exact` in norm: twice what
    the documented rounding of the operands costs on this input (other roundings
    of the same size fall elsewhere), the arithmetic, and the result's rounding."""
    t = 2 * rel(ns_emulated(g, dtype == torch.float32, **kw), exact)
    return t + ARITHMETIC + sums(max(g.shape[-2:])) + torch.finfo(dtype).eps / 2


def matrices(shape, seed, kind="spectrum", rms=1e-3):
    """A few strong directions over noise (a momentum's spectrum), or noise alone."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    if kind == "spectrum":
        r = max(1, min(shape[-2:]) // 8)
        left = torch.randn(*shape[:-1], r, generator=gen) / torch.arange(1, r + 1)
        x = left @ torch.randn(*shape[:-2], r, shape[-1], generator=gen) + 0.2 * x
    return x * rms
