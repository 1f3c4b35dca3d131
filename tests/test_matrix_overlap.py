"""Destinations (and Muon's parameters) that share elements are refused, whatever their
strides; ones that only interleave are taken."""
import ctypes

import pytest
import torch

import soar_b200 as sb
from matrix_helpers import matrices, ns64, rel, tolerance
from soar_b200 import optim
from test_muon import _create as create_muon
from test_ortho import _create

gpu = pytest.mark.gpu


def _dst(at, count, rows, cols, row, mat, src=1 << 30):
    """A stack into element `at` of one bf16 buffer."""
    return optim.MatrixDesc(src, (1 << 20) + 2 * at, count, rows, cols, row or cols, mat, row or cols, mat)


# of a buffer of rows of 100: rows 0 .. 9, columns from 0
FIRST = (0, 1, 10, 40, 100, 0)


@pytest.mark.parametrize("other", [
    (39, 1, 10, 40, 100, 0),          # one column shared
    (900 + 39, 1, 1, 1, 1, 0),        # its last element alone
    (500, 1, 400, 1, 1, 0),           # a column of ones that runs through its rows
    (40, 3, 10, 20, 100, 30),         # the third matrix reaches the next row
    (30, 2, 5, 40, 200, 100),         # interleaved matrices, ten columns shared
    (40, 1, 2, 61, 950, 0),           # its first row reaches into the second of the first one's
])
def test_refuses_overlapping_destinations(other):
    rc, why = _create([_dst(*FIRST), _dst(*other)])
    assert rc == -1 and "overlap" in why, why
    rc, why = _create([_dst(5000, 1, 3, 3, 0, 0), _dst(*other), _dst(2000, 1, 3, 3, 0, 0), _dst(*FIRST)])
    assert rc == -1 and "overlap" in why, why


@pytest.mark.parametrize("other", [
    (40, 1, 10, 60, 100, 0),          # the buffer's other columns
    (40, 3, 10, 20, 100, 20),         # the same, as a stack of column slices
    (940, 1, 10, 60, 60, 0),          # behind it
    (1000, 2, 5, 40, 200, 100),       # interleaved rows behind it
    (40, 1, 2, 60, 900, 0),           # two of the gaps between its rows
])
def test_takes_interleaved_destinations(other):
    rc, why = _create([_dst(*FIRST), _dst(*other)])
    assert rc == 0 or "overlap" not in why, why


def test_refuses_overlapping_parameters():
    def create(params, shapes):
        lib = sb.lib()
        o = optim.MuonOpts()
        lib.soar_muon_default_opts(ctypes.byref(o))
        k = len(shapes)
        t = (optim.TensorDesc * k)(*[optim.TensorDesc(p, 1 << 30, c * r * n, 0.0)
                                     for p, (c, r, n) in zip(params, shapes)])
        s = (optim.MatrixShape * k)(*[optim.MatrixShape(*q) for q in shapes])
        out = ctypes.c_void_p()
        rc = lib.soar_muon_create(t, s, k, ctypes.byref(o), ctypes.byref(out))
        return rc, lib.soar_last_error().decode()

    base = 1 << 20
    for at in (4, 4 * 31, -4 * 15):
        rc, why = create([base, base + (1 << 16), base + at], [(1, 4, 8), (1, 3, 3), (1, 4, 4)])
        assert rc == -1 and "overlap" in why, why
    assert create_muon([(1, 4, 8), (2, 4, 4)], [32, 32])[0] == -1


@gpu
def test_column_slices_of_one_buffer(cuda):
    """Interleaved destinations are each as if alone, and so are adjacent parameters."""
    buf = torch.full((300, 500), 7.0, device="cuda")
    cuts = [(0, 130), (130, 131), (131, 400), (403, 500)]
    gs = [matrices((300, b - a), a).cuda() for a, b in cuts]
    sb.Orthogonalizer(gs, [buf[:, a:b] for a, b in cuts]).run()
    for g, (a, b) in zip(gs, cuts):
        want = ns64(g)
        assert rel(buf[:, a:b], want) <= tolerance(g, want, torch.float32)
    assert bool((buf[:, 400:403] == 7).all())
    with pytest.raises(sb.SoarError, match="overlap"):
        sb.Orthogonalizer(gs[:2], [buf[:, 0:130], buf[:, 129:130]])
    flat = torch.zeros(64 * 64 + 32 * 48, device="cuda")
    ws = [flat[:64 * 64].view(64, 64), flat[64 * 64:].view(32, 48)]
    opt = sb.Muon(ws, sb.MuonOptions(lr=1.0, scale="none", nesterov=False), grads=[matrices(w.shape, 3).cuda() for w in ws])
    opt.step()
    for w, g in zip(ws, opt.grads):
        want = ns64(g)
        assert rel(-w, want) <= tolerance(g, want, torch.float32)
    with pytest.raises(sb.SoarError, match="overlap"):
        sb.Muon([ws[0], flat[64 * 63:64 * 63 + 64].view(8, 8)], grads=[w.clone() for w in (ws[0], ws[0][:1].view(8, 8))])
