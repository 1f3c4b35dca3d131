"""Matrices of at most 8 rows (or columns) with bf16 results: the roundings of their few
singular values do not average out, so their products need more than 11 bits."""
import pytest
import torch

import soar_b200 as sb
from matrix_helpers import COEF, matrices, ns64, rel

gpu = pytest.mark.gpu

# Before the result's rounding: X's start is held in 22 bits, so that it is off by at most 2^-22
# of a norm of 1. A step multiplies that by at most the coefficient a (its slope at 0, the
# largest in magnitude): 3.4445^5 < 485. The result's norm is at least 0.68, which the
# iteration takes its largest singular value to, and what follows has 64 bits.
HELD = 485 * 2.0 ** -22 / 0.68

SIDES = [(1, 1), (1, 2), (2, 1), (1, 7), (1, 515), (515, 1), (2, 2), (2, 3), (3, 2), (2, 64), (3, 3), (3, 64), (512, 3),
         (4, 4), (4, 5), (4, 9), (4, 512), (700, 4), (5, 300), (6, 6), (6, 48), (7, 5), (7, 1000), (8, 8), (8, 9),
         (9, 8), (8, 4097), (2048, 8), (1, 70000)]


def _run(g, dst, **kw):
    out = torch.full(g.shape, 7.0, dtype=dst, device="cuda")
    plan = sb.Orthogonalizer([g], [out], sb.OrthogonalizeOptions(**kw))
    plan.run()
    assert plan.error() == 0
    return out


def _close(got, want, held=HELD):
    """Elements within their own rounding to bf16 (2^-8), and what the held start is off by."""
    bound = want.abs() * 2.0 ** -8 + (1 + 2.0 ** -8) * held * want.square().sum(dim=(-2, -1), keepdim=True).sqrt()
    return bool(((got.double() - want).abs() <= bound).all())


@gpu
@pytest.mark.parametrize("shape", SIDES, ids=lambda s: f"{s[0]}x{s[1]}")
@pytest.mark.parametrize("src", [torch.float32, torch.bfloat16])
def test_bf16_results(cuda, shape, src):
    for seed in range(12):
        g = matrices(shape, 100 * seed + shape[0], "spectrum" if seed % 2 else "noise").to(src).cuda()
        want = ns64(g)
        assert _close(_run(g, torch.bfloat16), want), seed


@gpu
def test_stacks_strides_and_other_matrices(cuda):
    """Stacks of them in slices of larger buffers, beside matrices of more rows."""
    shapes = [(300, 3, 40), (5, 33, 8), (4, 100, 70), (2, 8, 700), (1, 300, 290), (170, 1, 1)]
    srcs, dsts, bufs = [], [], []
    for i, s in enumerate(shapes):
        x = torch.nn.functional.pad(matrices(s, 20 + i), (3, 2)).cuda()
        buf = torch.full_like(x, 7.0, dtype=torch.bfloat16)
        srcs.append(x[..., 3:-2])
        dsts.append(buf[..., 3:-2])
        bufs.append(buf)
    plan = sb.Orthogonalizer(srcs, dsts)
    for _ in range(2):
        plan.run()
    assert plan.error() == 0
    for s, x, y, buf in zip(shapes, srcs, dsts, bufs):
        assert bool((buf[..., :3] == 7).all()) and bool((buf[..., -2:] == 7).all())
        want = ns64(x)
        if min(s[1:]) <= 8:
            assert _close(y, want), s
        else:
            assert rel(y, want) <= 2.0 ** -7


@gpu
def test_values_and_steps(cuda):
    g = matrices((6, 5, 90), 3)
    g[0] = 0
    g[1, 4, 6] = float("inf")
    g[2, 0, 89] = float("nan")
    g[3] *= 1e-20
    g[4] = 1.0
    out = _run(g.cuda(), torch.bfloat16)
    assert bool((out[0] == 0).all()) and bool(out[1].isnan().all()) and bool(out[2].isnan().all())
    for i in (3, 4, 5):
        assert _close(out[i], ns64(g[i].cuda(), eps=float(torch.tensor(1e-7)))), i
    for steps in (1, 2, 12):
        # singular values that start above 0.3 are above 0.68 from the second step on, where a
        # step's slope is at most 1.9 in magnitude
        x = (torch.eye(5, 90) + 0.01 * matrices((5, 90), 4, "noise", 1.0)).cuda()
        held = HELD / 485 * 3.4445 ** min(steps, 2) * 1.9 ** max(steps - 2, 0)
        assert _close(_run(x, torch.bfloat16, steps=steps), ns64(x, steps=steps), held), steps
    coef = ((4.0, -6.0, 2.5), (3.0, -3.2, 1.2), (1.875, -1.25, 0.375))
    x = matrices((7, 31), 5).cuda()
    assert _close(_run(x, torch.bfloat16, steps=3, coefficients=coef), ns64(x, steps=3, coef=coef))


@gpu
def test_sources_that_are_others_destinations(cuda):
    """Two matrices that change places: every source is read before a result is written."""
    for shape in ((4, 300), (300, 4)):
        x = torch.stack([matrices(shape, k) for k in (1, 2)]).bfloat16().cuda()
        want = ns64(x).flip(0)
        sb.Orthogonalizer([x[0], x[1]], [x[1], x[0]]).run()
        assert _close(x, want)


@gpu
@pytest.mark.parametrize("ema", [False, True])
def test_mixed_muon(cuda, ema):
    """Weights of zero take the update itself; decay, factor and EMA as for any weight."""
    shapes = [(3, 100), (64, 8), (10, 2, 33), (1, 1), (100, 100)]
    grads = [matrices(s, i).bfloat16().cuda() for i, s in enumerate(shapes)]
    ws = [torch.zeros(s, dtype=torch.bfloat16, device="cuda") for s in shapes]
    opt = sb.Muon(ws, sb.MuonOptions(lr=0.5, momentum=0.0, nesterov=False, scale="none", weight_decay=0.25),
                  grads=grads, layout="bf16_mixed")
    if ema:
        opt.enable_ema(0.75)
    for _ in range(2):
        opt.step()
    assert opt.info().error == 0
    for i, (w, g) in enumerate(zip(ws, grads)):
        o = ns64(g)
        want = -0.5 * o * (1 + (1 - 0.5 * 0.25))
        master = opt.state(i, sb.STATE_MASTER).view(w.shape)
        assert torch.equal(w, master.bfloat16())
        if min(w.shape[-2:]) > 8:
            continue
        for k in range(w.shape[0] if w.dim() == 3 else 1):
            m, t = (master[k], want[k]) if w.dim() == 3 else (master, want)
            # (three roundings of 2^-24 a step)
            assert rel(m, t) <= HELD + 6 * 2.0 ** -24, i
        if ema:
            e = opt.state(i, sb.STATE_EMA).view(w.shape)
            after_one = -0.5 * o
            assert rel(e, 0.75 * 0.25 * after_one + 0.25 * want) <= HELD + 12 * 2.0 ** -24
