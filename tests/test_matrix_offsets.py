"""The matrix operators where an element's offset passes 32 bits: strides of the caller's
buffers, and the workspace of a long stack in both product kernels."""
import pytest
import torch

import soar_b200 as sb
from matrix_helpers import matrices, ns64, rel, tolerance
from test_muon import Model64, _check

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("shape,stride", [((3, 100, 130), (1 << 31, 130, 1)), ((1, 3, 290), (1, 1 << 31, 1)),
                                          ((2, 300, 270), (1 << 32, 270, 1))], ids=str)
def test_strides(cuda, shape, stride):
    """Between matrices, or between rows."""
    size = 1 + sum((n - 1) * s for n, s in zip(shape, stride))
    src, dst = (torch.empty(size, dtype=torch.bfloat16, device="cuda").as_strided(shape, stride) for _ in range(2))
    src.copy_(matrices(shape, 5))
    plan = sb.Orthogonalizer([src], [dst])
    plan.run()
    assert plan.error() == 0
    for k in range(shape[0]):
        want = ns64(src[k])
        assert rel(dst[k], want) <= tolerance(src[k].contiguous(), want, torch.bfloat16)
    del plan, src, dst
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("shape", [(14700, 256, 1152), (14100, 300, 1024)], ids=str)
def test_long_stack(cuda, shape):
    """A stack of more than 2^32 elements, in place."""
    x = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    edge = (1 << 32) // (shape[1] * shape[2])   # the matrix across the boundary
    assert edge + 1 < shape[0]
    at = (0, 1, edge - 1, edge, edge + 1, shape[0] - 1)
    before = {k: x[k].clone() for k in at}
    plan = sb.Orthogonalizer([x], [x])
    plan.run()
    assert plan.error() == 0
    for k, g in before.items():
        want = ns64(g)
        assert rel(x[k], want) <= tolerance(g, want, torch.bfloat16), k
    del plan, x
    torch.cuda.empty_cache()


@gpu
def test_mixed_layout_ema(cuda):
    """The weight EMA of mixed-precision Muon, in blocks of four and of odd elements."""
    shapes = [(64, 96), (70, 51), (300, 320), (2, 270, 261)]
    params = [matrices(s, i, "noise", 0.02).bfloat16().cuda() for i, s in enumerate(shapes)]
    grads = [matrices(s, 10 + i).bfloat16().cuda() for i, s in enumerate(shapes)]
    opts = sb.MuonOptions(lr=5e-3, weight_decay=0.1)
    opt = sb.Muon(params, opts, grads=grads, layout="bf16_mixed")
    opt.enable_ema(0.9)
    model = Model64(params, [0.1] * len(shapes), opts, ema=0.9)
    for _ in range(3):
        opt.step()
        model.step(grads, False)
    assert opt.info().error == 0
    _check(opt, model, params, True, 3)
    for i, p in enumerate(params):
        e = opt.state(i, sb.STATE_EMA).view(p.shape).double()
        # a mean of weights that are each within their bound, and three roundings a step
        bound = model.move[i] + 9 * 2.0 ** -23 * float(model.ema[i].norm())
        assert float((e - model.ema[i]).norm()) <= bound
