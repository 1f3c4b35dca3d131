"""Coefficients of the Newton-Schulz steps beyond fp16's range are refused; up to it they
give the definition's result."""
import pytest
import torch

import soar_b200 as sb
from matrix_helpers import matrices, ns64, rel, tolerance
from soar_b200 import optim
from test_muon import _create as create_muon
from test_ortho import _create as create_ortho
from test_ortho import _desc

gpu = pytest.mark.gpu


def _coef(*rows):
    rows = list(rows) + [(0.0, 0.0, 0.0)] * (optim.NS_MAX_STEPS - len(rows))
    return ((optim.C.c_float * 3) * optim.NS_MAX_STEPS)(*[(optim.C.c_float * 3)(*r) for r in rows])


@pytest.mark.parametrize("rows,word", [
    ([(8.0, 0.0, 0.0)], "7.99"),
    ([(3.0, 0.0, 0.0), (3.0, 0.0, 0.0)], "7.99"),            # 9 after two steps
    ([(1.0, 8.0, 0.0)], "7.99"),                             # by b alone
    ([(-9.0, 0.0, 0.0)], "7.99"),
    ([(61.0, -61.0, 0.0)], "60"),                            # B of small singular values
    ([(7.0, 0.0, 0.0), (1.0, 0.0, -0.026)], "60"),   # at a singular value of 7
    ([(float("nan"), 0.0, 0.0)], "finite"),
    ([(1.0, 0.0, float("inf"))], "finite"),
])
def test_refuses_coefficients_past_fp16(rows, word):
    over = {"steps": len(rows), "coef": _coef(*rows)}
    for rc, why in (create_ortho([_desc()], **over), create_muon([(1, 4, 8)], [32], **over)):
        assert rc == -1 and "coefficients" in why and word in why, why


@pytest.mark.parametrize("rows", [
    [(3.4445, -4.7750, 2.0315)] * 16, [(2.0, -1.5, 0.5)] * 5, [(1.5, -0.5, 0.0)] * 16, [(7.9, 0.0, 0.0)],
    [(15 / 8, -10 / 8, 3 / 8)] * 10, [(0.0, 0.0, 0.0)] * 3,
    # (steps behind the last are not looked at)
    [(4.0, -6.0, 2.5), (3.0, -3.2, 1.2)] + [(float("nan"), 0.0, 0.0)] * 2])
def test_takes_coefficients_within(rows):
    steps = 2 if rows[-1][0] != rows[-1][0] else len(rows)
    rc, why = create_ortho([_desc()], steps=steps, coef=_coef(*rows))
    assert rc == 0 or "coefficients" not in why, why


@gpu
@pytest.mark.parametrize("shape", [(90, 120), (270, 300)], ids=str)
def test_results_up_to_the_bound(cuda, shape):
    """Singular values of up to 7.9, whole matrices and tile by tile."""
    gen = torch.Generator().manual_seed(3)
    g = torch.randn(shape[0], 1, generator=gen) @ torch.randn(1, shape[1], generator=gen) + 0.01 * matrices(shape, 4, rms=1.0)
    coef = ((7.9, 0.0, 0.0), (0.1, 0.001, 0.0001))
    for dst in (torch.float32, torch.bfloat16):
        out = torch.empty(shape, dtype=dst, device="cuda")
        x = g.cuda()
        sb.Orthogonalizer([x], [out], sb.OrthogonalizeOptions(steps=2, coefficients=coef)).run()
        want = ns64(x, steps=2, coef=coef)
        assert rel(out, want) <= tolerance(x, want, dst, steps=2, coef=coef)
