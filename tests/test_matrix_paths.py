"""The matrix operators on lists long enough for the tiles, preparation tiles and
lists of matrices that large workloads use, against the definition in 64 bits:
256-column tiles of every product (mirrored ones among them), preparation tiles
of four squares of matrices with more rows than columns and of Muon's, operands
of more than one list of 256 MB, and fp32 results of sides beyond 1024."""
import pytest
import torch

import soar_b200 as sb
from matrix_helpers import matrices, ns64, rel, tolerance
from test_muon import Model64, _check

gpu = pytest.mark.gpu


def _symmetric_tiles(shapes, wide):
    """Tiles of X X^T and A A: 256 rows by `wide` columns, on and right of the diagonal's blocks."""
    total = 0
    for count, r, c in shapes:
        m = min(r, c)
        total += count * sum(-(-(m - top) // wide) for top in range(0, m, 256))
    return total


def _squares(shapes):
    return sum(n * -(-r // 64) * -(-c // 64) for n, r, c in shapes)


def _operand_bytes(shapes, fp32):
    up = lambda x, a: -(-x // a) * a  # noqa: E731
    return sum(n * min(r, c) * ((8 if fp32 else 6) * up(max(r, c), 64) + (8 if fp32 else 4) * up(min(r, c), 8))
               for n, r, c in shapes)


def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def _orthogonalized(shapes, seed, dst, src=torch.float32):
    gs = [matrices(s, seed + i).to(src).cuda() for i, s in enumerate(shapes)]
    out = [torch.full(s, 7.0, dtype=dst, device="cuda") for s in shapes]
    plan = sb.Orthogonalizer(gs, out)
    plan.run()
    assert plan.error() == 0
    return gs, out


def _compare(gs, out, dst):
    for i, (g, o) in enumerate(zip(gs, out)):
        for k in range(g.shape[0]):
            want = ns64(g[k])
            assert rel(o[k], want) <= tolerance(g[k], want, dst), (i, k)


# X X^T and A A of three tiles a matrix and more, the third or so mirrored; wide, tall, odd
WIDE = [(20, 512, 520), (16, 515, 700), (12, 700, 513), (4, 1000, 600), (3, 770, 1030), (2, 1100, 300)]


@gpu
@pytest.mark.parametrize("src", [torch.float32, torch.bfloat16])
def test_wide_tiles(cuda, src):
    assert _symmetric_tiles(WIDE, 256) >= _sms() // 2 and _squares(WIDE) >= 16 * _sms()
    _compare(*_orthogonalized(WIDE, 300, torch.bfloat16, src), torch.bfloat16)


@gpu
def test_long_lists_of_at_most_256_rows(cuda):
    """Whole matrices on a pair of CTAs each, more of them than pairs, tall and wide."""
    shapes = [(90, 300, 200), (60, 256, 640), (30, 1000, 129), (8, 64, 64)]
    assert _squares(shapes) >= 16 * _sms()
    _compare(*_orthogonalized(shapes, 320, torch.bfloat16), torch.bfloat16)


@gpu
@pytest.mark.parametrize("dst", [torch.bfloat16, torch.float32])
def test_operands_of_several_lists(cuda, dst):
    shapes = [(40, 1024, 1024), (12, 1300, 1100), (9, 600, 2000), (30, 200, 300)]
    assert _operand_bytes(shapes[:3], dst == torch.float32) >= 2 * (256 << 20)
    _compare(*_orthogonalized(shapes, 340, dst), dst)


@gpu
@pytest.mark.parametrize("shape", [(1, 1500, 1900), (1, 2048, 1300)], ids=str)
def test_fp32_results_of_long_sides(cuda, shape):
    _compare(*_orthogonalized([shape], 360, torch.float32), torch.float32)


@gpu
@pytest.mark.parametrize("layout,shapes", [("bf16_mixed", WIDE), ("fp32", WIDE),
                                           ("bf16_mixed", [(90, 300, 200), (60, 256, 640), (8, 64, 64)])])
def test_muon_long_lists(cuda, layout, shapes):
    mixed = layout == "bf16_mixed"
    dt = torch.bfloat16 if mixed else torch.float32
    params = [matrices(s, i, "noise", 0.02).to(dt).cuda() for i, s in enumerate(shapes)]
    grads = [matrices(s, 400 + i).to(dt).cuda() for i, s in enumerate(shapes)]
    opts = sb.MuonOptions(lr=2e-3, scale="rms", weight_decay=0.1)
    opt = sb.Muon(params, opts, grads=grads, layout=layout)
    # matrix by matrix: an error in one is not lost among the others of its stack
    model = [Model64([p[k] for p in params for k in range(p.shape[0])],
                     [0.1] * sum(p.shape[0] for p in params), opts)]
    flat = [g[k] for g in grads for k in range(g.shape[0])]
    for _ in range(2):
        opt.step()
        model[0].step(flat, not mixed)
    assert opt.info().error == 0

    class Views:
        """The optimizer's state, matrix by matrix."""

        def __init__(self):
            self.at = [(i, k) for i, p in enumerate(params) for k in range(p.shape[0])]

        def state(self, index, kind):
            i, k = self.at[index]
            return opt.state(i, kind).view(params[i].shape)[k].reshape(-1)

    _check(Views(), model[0], [p[k] for p in params for k in range(p.shape[0])], mixed, 2)
