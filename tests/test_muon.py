"""Muon on the fused device step (soar_muon_create): refusals (no GPU), and the
whole step against its definition in 64 bits: momentum, skip and loss-scale
sequence, clip, shape factors, weight decay, EMA, gradient sets, checkpoint,
capture, beside an AdamW."""
import ctypes
import math

import numpy as np
import pytest
import torch

import soar_b200 as sb
from matrix_helpers import ARITHMETIC, matrices, ns64, ns_emulated, rel, sums
from soar_b200 import optim

gpu = pytest.mark.gpu


def _create(shapes, numels, n=None, **over):
    lib = sb.lib()
    o = optim.MuonOpts()
    lib.soar_muon_default_opts(ctypes.byref(o))
    for k, v in over.items():
        setattr(o, k, v)
    k = len(shapes)
    t = (optim.TensorDesc * k)(*[optim.TensorDesc(4096, 8192, m, 0.0) for m in numels])
    s = (optim.MatrixShape * k)(*[optim.MatrixShape(*q) for q in shapes])
    out = ctypes.c_void_p()
    rc = lib.soar_muon_create(t, s, k, ctypes.byref(o), ctypes.byref(out))
    return rc, lib.soar_last_error().decode()


@pytest.mark.parametrize("shape,numel,over,word", [
    ((1, 4, 8), 31, {}, "numel"),
    ((2, 4, 8), 32, {}, "numel"),
    ((1, (1 << 20) + 1, 1), (1 << 20) + 1, {}, "1048576"),
    ((1, 4, 8), 32, {"steps": 0}, "steps"),
    ((1, 4, 8), 32, {"steps": 17}, "steps"),
    ((1, 4, 8), 32, {"scale": 3}, "scale"),
    ((1, 4, 8), 32, {"eps": -1.0}, "eps"),
    ((1, 4, 8), 32, {"layout": 7}, "layout"),
])
def test_refusals(shape, numel, over, word):
    rc, why = _create([shape], [numel], **over)
    assert rc == -1 and word in why, why


def test_refuses_the_same_parameters_twice():
    rc, why = _create([(1, 4, 8), (2, 4, 4)], [32, 32])
    assert rc == -1 and "same parameters" in why, why


def test_null_arguments_and_defaults():
    lib = sb.lib()
    out = ctypes.c_void_p()
    assert lib.soar_muon_create(None, None, 1, None, ctypes.byref(out)) == -1
    o = optim.MuonOpts()
    lib.soar_muon_default_opts(ctypes.byref(o))
    d = sb.MuonOptions()
    f = lambda v: ctypes.c_float(v).value  # noqa: E731
    assert (o.lr, o.momentum, bool(o.nesterov), o.weight_decay, o.steps, o.eps) == (
        f(d.lr), f(d.momentum), d.nesterov, f(d.weight_decay), d.steps, f(d.eps))
    assert optim.MUON_SCALES[d.scale] == o.scale
    assert all(o.coef[i][j] == f(d.coefficients[j]) for i in range(16) for j in range(3))


def test_python_refusals():
    w = torch.zeros(4, 8)
    for bad, word in ((torch.zeros(8), "rows, cols"), (torch.zeros(1, 2, 3, 4), "rows, cols"),
                      (w.t(), "contiguous")):
        with pytest.raises(ValueError, match=word):
            sb.Muon([bad], grads=[bad])
    with pytest.raises(ValueError, match="scale"):
        sb.Muon([w], sb.MuonOptions(scale="width"), grads=[w])


def test_structs_match_the_c_layout(tmp_path):
    """Sizes and offsets of the structs of the matrix operators, as a C compiler has them."""
    import shutil
    import subprocess
    from pathlib import Path
    cc = shutil.which("gcc") or shutil.which("cc")
    if not cc:
        pytest.skip("no C compiler")
    pairs = [("soar_matrix_desc", optim.MatrixDesc), ("soar_ortho_opts", optim.OrthoOpts),
             ("soar_matrix_shape", optim.MatrixShape), ("soar_muon_opts", optim.MuonOpts)]
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "soar_optim.h"', "int main(void) {"]
    want = []
    for name, py in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(py))
        for f, _ in py._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {f}));')
            want.append(getattr(py, f).offset)
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text("\n".join([*lines, "return 0; }"]))
    inc = Path(__file__).resolve().parents[1] / "include"
    subprocess.run([cc, "-std=c99", "-I", str(inc), str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == want


# ----------------------------------------------------------------------------

def _factor(scale, rows, cols):
    return {"none": 1.0, "aspect": math.sqrt(max(1.0, rows / cols)),
            "rms": 0.2 * math.sqrt(max(rows, cols))}[scale]


class Model64:
    """The step's definition in 64 bits (scaler decisions as the library's)."""

    def __init__(self, params, wd, opts, max_norm=0.0, scale=None, interval=200, ema=None):
        self.w = [p.double().clone() for p in params]
        self.m = [torch.zeros_like(w) for w in self.w]
        self.wd, self.o, self.max_norm = wd, opts, max_norm
        self.scale, self.interval, self.tracker = scale, interval, 0
        self.t = self.skipped = 0
        self.ema, self.decay = ([w.clone() for w in self.w] if ema else None), ema
        self.move = [0.0] * len(self.w)   # what the steps' directions may be off by, summed

    def step(self, grads, three):
        inv = 1.0 / self.scale if self.scale else 1.0
        gs = [None if g is None else g.double() * inv for g in grads]
        total = sum(float(g.square().sum()) for g in gs if g is not None)
        if self.scale and not math.isfinite(total):
            self.skipped += 1
            self.scale *= 0.5
            self.tracker = 0
            return
        norm = math.sqrt(total)
        coef = self.max_norm / norm if self.max_norm and norm > self.max_norm else 1.0
        self.t += 1
        if self.scale:
            self.tracker += 1
            if self.tracker == self.interval:
                self.scale *= 2
                self.tracker = 0
        for i, g in enumerate(gs):
            if g is None:
                continue
            d = g * coef
            self.m[i] = self.o.momentum * self.m[i] + d
            u = d + self.o.momentum * self.m[i] if self.o.nesterov else self.m[i]
            o = ns64(u, steps=self.o.steps)
            s = self.o.lr * _factor(self.o.scale, *u.shape[-2:])
            off = 2 * rel(ns_emulated(u, three, steps=self.o.steps), o) + ARITHMETIC + sums(max(u.shape[-2:]))
            self.move[i] += s * off * float(o.norm())
            self.w[i] = self.w[i] * (1.0 - self.o.lr * self.wd[i]) - s * o
            if self.ema:
                self.ema[i] = self.decay * self.ema[i] + (1 - self.decay) * self.w[i]


def _check(opt, model, params, mixed, steps):
    for i, p in enumerate(params):
        w = model.w[i]
        master = opt.state(i, sb.STATE_MASTER).view(p.shape).double()
        # the directions, and three roundings a step of the weights (the decay's product
        # and difference, the update's), each of at most half a step
        bound = model.move[i] + 3 * steps * 2.0 ** -24 * float(w.norm())
        err = float((master - w).norm())
        assert err <= bound, (i, err, bound)
        if mixed:  # the parameters are the master weights, rounded
            assert torch.equal(p, opt.state(i, sb.STATE_MASTER).view(p.shape).bfloat16())
        mom = opt.state(i, sb.STATE_M).view(p.shape)
        # a step rounds the clip's product, the decay's and the sum
        assert rel(mom, model.m[i]) <= 4 * steps * 2.0 ** -24, i


SHAPES = [(64, 64), (3, 40, 72), (130, 257), (300, 96), (1, 33), (17, 1), (2, 128, 512)]


@gpu
@pytest.mark.parametrize("layout,scale,nesterov,wd,clip,scaler", [
    ("fp32", "aspect", True, 0.1, 0.0, False), ("fp32", "none", False, 0.0, 0.5, False),
    ("fp32", "rms", True, 0.05, 0.0, True), ("bf16_mixed", "rms", True, 0.1, 1.0, True),
    ("bf16_mixed", "aspect", False, 0.0, 0.0, False), ("bf16_mixed", "none", True, 0.1, 0.0, True)])
def test_steps_match_definition(cuda, layout, scale, nesterov, wd, clip, scaler):
    mixed = layout == "bf16_mixed"
    dt = torch.bfloat16 if mixed else torch.float32
    params = [(matrices(s, i, "noise", 0.02)).to(dt).cuda() for i, s in enumerate(SHAPES)]
    grads = [torch.empty_like(p) for p in params]
    opts = sb.MuonOptions(lr=2e-3, scale=scale, nesterov=nesterov, weight_decay=wd)
    opt = sb.Muon([sb.ParamGroup(params[:4], wd), sb.ParamGroup(params[4:], 0.0)], opts, grads=grads,
                  layout=layout, max_grad_norm=clip,
                  loss_scaler=sb.LossScalerOptions(init_scale=1024.0, growth_interval=3) if scaler else None)
    assert opt.kernel_path == "matrix"
    model = Model64(params, [wd] * 4 + [0.0] * 3, opts, clip, 1024.0 if scaler else None, 3)
    steps = 7
    for t in range(steps):
        for i, g in enumerate(grads):
            g.copy_(matrices(g.shape, 100 * t + i, rms=1e-2 * (model.scale or 1.0)))
        if scaler and t == 3:
            grads[2][7, 9] = float("inf")
        model.step(grads, not mixed)
        opt.step()
        info = opt.info()
        assert info.error == 0
        assert (info.step, info.skipped) == (model.t, model.skipped)
        if scaler:
            assert info.loss_scale == model.scale and info.growth_tracker == model.tracker
    _check(opt, model, params, mixed, steps)


@gpu
@pytest.mark.parametrize("layout", ["fp32", "bf16_mixed"])
def test_parameters_at_odd_offsets(cuda, layout):
    """Parameters and gradients that start one to three elements into a buffer:
    the elements around them stay, and the step is the same."""
    dt = torch.bfloat16 if layout == "bf16_mixed" else torch.float32
    shapes = [(64, 64), (64, 128), (300, 96), (260, 520), (2, 32, 64)]

    def place(x, off):
        buf = torch.full((x.numel() + 8,), 7.0, dtype=dt, device="cuda")
        buf[off:off + x.numel()] = x.to(dt).cuda().flatten()
        return buf, buf[off:off + x.numel()].view(x.shape)

    ps = [place(matrices(s, i, "noise", 0.02), 1 + i % 3) for i, s in enumerate(shapes)]
    gs = [place(matrices(s, 50 + i), 1 + i % 3) for i, s in enumerate(shapes)]
    params = [v for _, v in ps]
    opts = sb.MuonOptions(lr=2e-3, scale="rms", weight_decay=0.1)
    opt = sb.Muon(params, opts, grads=[v for _, v in gs], layout=layout)
    model = Model64(params, [0.1] * len(shapes), opts)
    for _ in range(2):
        model.step([v for _, v in gs], layout == "fp32")
        opt.step()
    assert opt.info().error == 0
    _check(opt, model, params, layout == "bf16_mixed", 2)
    for i, (buf, v) in enumerate(ps + gs):
        off = 1 + i % len(shapes) % 3
        assert bool((buf[:off] == 7).all()) and bool((buf[off + v.numel():] == 7).all())


@gpu
def test_large_weight(cuda):
    """Many tiles in every product, in both layouts."""
    for layout, dt in (("fp32", torch.float32), ("bf16_mixed", torch.bfloat16)):
        w = matrices((900, 1300), 1, "noise", 0.02).to(dt).cuda()
        g = matrices((900, 1300), 2).to(dt).cuda()
        opts = sb.MuonOptions(lr=1e-3, scale="rms", weight_decay=0.1)
        opt = sb.Muon([w], opts, grads=[g], layout=layout)
        model = Model64([w], [0.1], opts)
        for _ in range(2):
            model.step([g], layout == "fp32")
            opt.step()
        assert opt.info().error == 0
        _check(opt, model, [w], layout != "fp32", 2)


@gpu
def test_clip_calls_and_partial_sums(cuda):
    """clip_grad_norm, its asynchronous form and grad_sumsq / apply take the same step as
    max_grad_norm does."""
    def make(**kw):
        w = matrices((2, 96, 130), 1, "noise", 0.02).bfloat16().cuda()
        g = matrices((2, 96, 130), 2, rms=1.0).bfloat16().cuda()
        return w, sb.Muon([w], sb.MuonOptions(lr=1e-3), grads=[g], layout="bf16_mixed", **kw)

    w0, a = make(max_grad_norm=0.25)
    a.step()
    w1, b = make()
    norm = b.clip_grad_norm(0.25)
    b.step()
    w2, c = make()
    c.clip_grad_norm_async(0.25)
    c.step()
    w3, d = make(max_grad_norm=0.25)
    part = torch.zeros(1, dtype=torch.float64, device="cuda")
    d.grad_sumsq(part.data_ptr())
    d.apply(part.data_ptr(), 1)
    assert norm == a.info().grad_norm
    for w, o in ((w1, b), (w2, c), (w3, d)):
        assert torch.equal(w, w0) and o.info().clip_coef < 1
        assert torch.equal(o.state(0, sb.STATE_M), a.state(0, sb.STATE_M))


@gpu
def test_ema_sets_and_missing_gradients(cuda):
    shapes = [(48, 80), (100, 60), (33, 33)]
    params = [matrices(s, i, "noise", 0.02).cuda() for i, s in enumerate(shapes)]
    sets = [[matrices(s, 10 * k + i).cuda() for i, s in enumerate(shapes)] for k in range(2)]
    for s in sets:
        s[1] = None
    opts = sb.MuonOptions(lr=5e-3)
    opt = sb.Muon(params, opts, grads=sets[0])
    assert opt.add_grads(sets[1]) == 1
    opt.enable_ema(0.9)
    model = Model64(params, [0.0] * 3, opts, ema=0.9)
    before = params[1].clone()
    for t in range(4):
        opt.use_grads(t & 1)
        opt.step()
        model.step(sets[t & 1], True)
    _check(opt, model, params, False, 4)
    assert torch.equal(params[1], before)
    for i in (0, 2):
        e = opt.state(i, sb.STATE_EMA).view(params[i].shape).double()
        # a mean of weights that are each within their bound, and three roundings a step
        bound = model.move[i] + 24 * 2.0 ** -24 * float(model.ema[i].norm())
        assert float((e - model.ema[i]).norm()) <= bound
    opt.zero_grad()
    assert bool((sets[1][0] == 0).all())
    with pytest.raises(sb.SoarError, match="second-moment"):
        opt.read_state(0, sb.STATE_V)


@gpu
def test_checkpoint_resumes_bit_for_bit(cuda, tmp_path):
    shapes = [(70, 50), (2, 64, 96)]

    def make():
        ps = [matrices(s, i, "noise", 0.02).bfloat16().cuda() for i, s in enumerate(shapes)]
        gs = [torch.empty_like(p) for p in ps]
        return ps, gs, sb.Muon(ps, sb.MuonOptions(lr=1e-3, weight_decay=0.1), grads=gs,
                               layout="bf16_mixed", loss_scaler=sb.LossScalerOptions(init_scale=64.0))

    def go(gs, opt, t):
        for i, g in enumerate(gs):
            g.copy_(matrices(g.shape, 50 * t + i, rms=1.0))
        if t == 1:
            gs[0][3, 3] = float("nan")
        opt.step()

    ps, gs, opt = make()
    for t in range(5):
        go(gs, opt, t)
        if t == 2:
            opt.save_state(tmp_path / "muon.soar")
    qs, hs, other = make()
    other.load_state(tmp_path / "muon.soar")
    for t in range(3, 5):
        go(hs, other, t)
    assert opt.info().as_dict() == other.info().as_dict()
    for i, (p, q) in enumerate(zip(ps, qs)):
        assert torch.equal(p, q)
        for kind in (sb.STATE_MASTER, sb.STATE_M):
            np.testing.assert_array_equal(opt.read_state(i, kind), other.read_state(i, kind))
    adam = sb.AdamW(ps, grads=gs, layout="bf16_mixed")
    with pytest.raises(sb.SoarError, match="different"):
        adam.load_state(tmp_path / "muon.soar")


@gpu
def test_capture_beside_adamw_and_schedule(cuda):
    """As a training loop uses it: Muon for the weights, AdamW for the biases, one cosine
    schedule each, both steps in one captured graph."""
    def make():
        w = [matrices((128, 200), 1, "noise", 0.02).cuda(), matrices((60, 60), 2, "noise", 0.02).cuda()]
        b = [torch.zeros(200, device="cuda")]
        gw = [matrices(p.shape, 5 + i).cuda() for i, p in enumerate(w)]
        gb = [torch.full_like(b[0], 1e-3)]
        return (w, b, gw, gb, sb.Muon(w, sb.MuonOptions(lr=1e-3), grads=gw, max_grad_norm=1.0),
                sb.AdamW(b, sb.AdamWOptions(lr=1e-3), grads=gb))

    w, b, gw, gb, muon, adam = make()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        muon.step()
        adam.step()
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    w2, b2, _, _, muon2, adam2 = make()
    for _ in range(4):
        muon2.step()
        adam2.step()
    torch.cuda.synchronize()
    assert muon.info().step == muon2.info().step == 4
    for p, q in zip(w + b, w2 + b2):
        assert torch.equal(p, q)
    sched = sb.CosineAnnealingLR(muon2, total_steps=10, eta_min=1e-5)
    sched.step()
    assert muon2.get_lr() < 1e-3


@gpu
def test_gathered_momentum_is_the_same_step(cuda):
    """A user who keeps the momentum elsewhere: Orthogonalizer on it gives the update that
    Muon's own step makes, to the rounding of the weights."""
    w = matrices((2, 150, 220), 3, "noise", 0.02).cuda()
    start = w.clone()
    g = matrices((2, 150, 220), 4).cuda()
    lr = 1e-2
    sb.Muon([w], sb.MuonOptions(lr=lr, scale="none", nesterov=False), grads=[g]).step()
    o = torch.empty_like(w)
    sb.Orthogonalizer([g], [o]).run()
    torch.cuda.synchronize()
    assert float(((start - lr * o) - w).abs().max()) <= 2.0 ** -23 * float(w.abs().max())


@gpu
def test_zero1_refuses_muon(cuda):
    w = torch.zeros(8, 8, dtype=torch.bfloat16, device="cuda")
    opt = sb.Muon([w], grads=[w.clone()], layout="bf16_mixed")
    base = (ctypes.c_void_p * 1)(w.data_ptr())
    out = ctypes.c_void_p()
    rc = sb.lib().soar_zero1_create(opt.handle, 0, 1, base, base, None, 0, ctypes.byref(out))
    assert rc == -1 and b"matrices" in sb.lib().soar_last_error()


@gpu
def test_state_view_keeps_the_optimizer(cuda):
    """The memory of a state view is the optimizer's: it stays while the view does."""
    import gc
    import weakref
    w = matrices((64, 64), 1, "noise", 0.02).cuda()
    opt = sb.Muon([w], grads=[w.clone()])
    opt.step()
    view, alive = opt.state(0, sb.STATE_M).view(64, 64), weakref.ref(opt)
    del opt
    gc.collect()
    assert alive() is not None
    assert bool((view == view).all())
    del view
    gc.collect()
    assert alive() is None
