"""The matrix operators where a matrix's norm is no larger than eps: X = G / (|G| + eps)
then starts far below a norm of 1, and its fp16 parts have to hold it all the same."""
import math

import pytest
import torch

import soar_b200 as sb
from matrix_helpers import COEF, matrices, ns64, rel, sums

gpu = pytest.mark.gpu

EPS = float(torch.tensor(1e-7))  # the default, as the library's 32 bits have it


def _lift(bound):
    """X of singular values up to `bound` is held 2^lift times larger: up to 1/2 .. 1."""
    return 0 if not bound < 0.5 else min(100, -math.frexp(bound)[1])


def emulated(g, three, steps=5, coef=COEF, eps=EPS):
    """The documented arithmetic (matrix_helpers.ns_emulated) with X held, before every step,
    by a power of two that its bound on the singular values allows. g: one matrix."""
    a, b, c = coef
    x = g.double()
    x = x if x.shape[0] <= x.shape[1] else x.t()
    m, n = x.shape
    sx = 2.0 ** min(12, max(6, math.floor(0.5 * math.log2(m * n))))
    norm = float(x.square().sum().sqrt())
    bound = norm / (norm + eps) if norm else 0.0
    hold = sx * 2.0 ** _lift(bound)
    x = x * (hold / (norm + eps)) if norm else x

    def parts(v):
        hi = v.float().half().double()
        return hi, (v - hi).float().half().double()

    def product(p, q):
        (ph, pl), (qh, ql) = p, q
        return ph @ qh + (ph @ ql + pl @ qh if three else 0.0)

    for _ in range(steps):
        xs = parts(x)
        ps = parts(product(xs, (xs[0].t(), xs[1].t())) * (1024 / hold / hold))
        held = ps[0] + ps[1] if three else ps[0]
        bs = parts(b * held + (c / 1024) * product(ps, ps))
        bound = min(bound * (abs(a) + abs(b) * bound ** 2 + abs(c) * bound ** 4), 1e9)
        now = sx * 2.0 ** _lift(bound)
        x = (a * (xs[0] + xs[1]) + product(bs, xs) / 1024) * (now / hold)
        hold = now
    x = x / hold
    return x if g.shape[0] <= g.shape[1] else x.t()


def tolerance(g, exact, dtype, steps=5, eps=EPS):
    """As matrix_helpers.tolerance: twice the documented roundings, 32-bit arithmetic, sums, the
    result's rounding. A step's arithmetic (44 x 2^-24) is multiplied by at most 1.71 by each later
    step, of which at most five leave the range where the step only multiplies by a."""
    arithmetic = 44 * 2.0 ** -24 * sum(1.71 ** min(k, 5) for k in range(steps))
    t = 2 * rel(emulated(g, dtype == torch.float32, steps=steps, eps=eps), exact)
    return t + arithmetic + sums(max(g.shape)) + torch.finfo(dtype).eps / 2


def _of_norm(shape, norm, seed):
    g = matrices(shape, seed)
    return (g.double() * (norm / float(g.double().norm()))).float()


def _run(g, dst, **kw):
    out = torch.full(g.shape, 7.0, dtype=dst, device="cuda")
    plan = sb.Orthogonalizer([g.cuda()], [out], sb.OrthogonalizeOptions(**kw))
    plan.run()
    assert plan.error() == 0
    return out


def test_emulation_is_the_definition():
    """The emulation without roundings that matter: what the tolerances rest on (CPU)."""
    for norm in (1.0, 1e-8, 1e-12, 1e-20):
        g = _of_norm((24, 40), norm, 1)
        want = ns64(g, eps=EPS)
        # 22 bits of X and of the products' operands, as for a norm of 1
        assert rel(emulated(g, True), want) <= 2e-6, norm


# the second shape goes tile by tile, the others whole where one product is enough
@gpu
@pytest.mark.parametrize("shape", [(96, 160), (300, 280), (200, 70)], ids=lambda s: f"{s[0]}x{s[1]}")
@pytest.mark.parametrize("dst", [torch.float32, torch.bfloat16])
def test_norms_around_and_below_eps(cuda, shape, dst):
    for norm in (1e-6, 2e-7, 1e-7, 1e-8, 1e-9, 1e-10, 1e-12, 1e-14, 1e-18, 1e-24, 1e-30):
        g = _of_norm(shape, norm, 7)
        want = ns64(g, eps=EPS)
        got = _run(g, dst).cpu()
        assert rel(got, want) <= tolerance(g, want, dst), (norm, rel(got, want))


@gpu
@pytest.mark.parametrize("dst", [torch.float32, torch.bfloat16])
def test_large_eps_and_many_steps(cuda, dst):
    """A caller's own eps above the norm; as many steps as lift such a matrix to norms around 1."""
    for shape in ((96, 160), (300, 280)):
        for norm, eps, steps in ((1e-6, 1e-2, 5), (1.0, 100.0, 5), (1e-12, 1e-7, 12), (1e-3, 1.0, 9)):
            g = _of_norm(shape, norm, 9)
            e = float(torch.tensor(eps))
            want = ns64(g, steps=steps, eps=e)
            got = _run(g, dst, steps=steps, eps=eps).cpu()
            assert rel(got, want) <= tolerance(g, want, dst, steps, e), (shape, norm, eps, rel(got, want))


@gpu
@pytest.mark.parametrize("dst", [torch.float32, torch.bfloat16])
def test_eps_of_zero(cuda, dst):
    """Zeros give zeros; a matrix of the smallest numbers is normalised like any other."""
    g = matrices((5, 80, 96), 3)
    g[0] = 0
    g[2] *= 1e-33
    g[3] = 0
    g[3, 5, 7] = 2.0 ** -149
    g[4] *= 1e30
    out = _run(g, dst, eps=0.0).cpu()
    assert bool((out[0] == 0).all())
    for i in (1, 2, 3, 4):
        want = ns64(g[i], eps=0.0)
        assert rel(out[i], want) <= tolerance(g[i], want, dst, eps=0.0), i


@gpu
def test_small_and_large_matrices_of_one_stack(cuda):
    """Each matrix of a stack is held by its own power of two, in both product kernels."""
    for shape in ((6, 64, 300), (6, 290, 270)):
        g = torch.stack([_of_norm(shape[1:], 10.0 ** -e, e) for e in (0, 6, 8, 11, 17, 25)])
        for dst in (torch.float32, torch.bfloat16):
            out = _run(g, dst).cpu()
            for i in range(shape[0]):
                want = ns64(g[i], eps=EPS)
                assert rel(out[i], want) <= tolerance(g[i], want, dst), i


@gpu
@pytest.mark.parametrize("layout", ["fp32", "bf16_mixed"])
def test_muon_of_tiny_gradients(cuda, layout):
    """A weight whose gradients have all but vanished moves as the definition says."""
    dt = torch.float32 if layout == "fp32" else torch.bfloat16
    for shape in ((64, 64), (300, 270)):
        g = _of_norm(shape, 1e-12, 4).to(dt)
        # weights of zero: they are the update, whose size then hides nothing
        w = torch.zeros(shape, dtype=dt, device="cuda")
        opt = sb.Muon([w], sb.MuonOptions(lr=1.0, momentum=0.0, nesterov=False, scale="none"),
                      grads=[g.cuda()], layout=layout)
        opt.step()
        master = opt.state(0, sb.STATE_MASTER).view(shape).cpu()
        want = ns64(g.float(), eps=EPS)
        kind = torch.float32 if layout == "fp32" else torch.bfloat16  # which products are taken
        assert rel(-master, want) <= tolerance(g.float(), want, kind)
