"""The matrix operators of the optimizer library and the sizes they are timed at.

Two operators, each on a list of stacks of matrices (a stack [count, rows, cols]
holds `count` matrices that are treated one by one):

  orthogonalize  O = NS(G): G / (|G|_F + eps), then `steps` times
                 A = X X^T, X <- a X + (b A + c A A) X (on the shorter side).
  muon_step      one step of the Muon optimizer: unscale by the loss scale, global
                 norm, skip on inf/NaN, clip, momentum m <- mu m + g, u = g + mu m
                 (Nesterov) or m, O = NS(u), w <- w - lr wd w - lr s O with s by the
                 matrix's shape, bf16 write-back of the fp32 master weights.

`run` computes them with elementary torch operations in 32 bits, or, where `own`
is true, by the library's entry points. `exact` computes them in 64 bits.
"""
import math
import sys
from pathlib import Path

import torch

own = False

NS = (3.4445, -4.7750, 2.0315)  # the quintic's coefficients, the library's default
STEPS = 5
EPS = 1e-7
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}

# The 48 pointwise convolutions [4C, C] of the segmentation-net tensor list
# (C cycles 32, 64, 128, 256, 512), tensors of equal shape stacked.
SEGNET = "10x128x32 10x256x64 10x512x128 9x1024x256 9x2048x512"
# Tensors of 16K to 256K elements as in the mixed-precision list of 400 (46M
# parameters), as matrices of many shapes, equal ones stacked.
RAGGED = ("24x128x131 24x130x192 24x200x160 24x96x512 24x256x200 24x250x257 24x384x192 24x192x448 "
          "24x320x320 24x300x400 24x512x250 24x256x544 24x640x240 24x400x400 24x416x416 24x512x400 "
          "16x480x480 16x512x512")
# 200M parameters in layers 1024 wide: sixteen of four square projections and the
# two matrices of a feed-forward block four times as wide.
LAYERS = "64x1024x1024 16x4096x1024 16x1024x4096"


def listed():
    ortho = {"op": "orthogonalize", "pad": 0}
    muon = {"op": "muon_step", "momentum": 0.95, "nesterov": True, "wd": 0.1, "scale": "rms",
            "clip": 0.0, "scaler": False, "lr": 2e-4}
    return [
        # one small weight: what a call costs at the least
        {"name": "ortho 1x64x64 bf16", **ortho, "shapes": "1x64x64", "src": "bf16", "dst": "bf16"},
        # the convolutions of the segmentation net, momentum and result in fp32
        {"name": "ortho segnet fp32", **ortho, "shapes": SEGNET, "src": "fp32", "dst": "fp32"},
        # odd sizes, a row, a column and padded rows, as slices of larger buffers are
        {"name": "ortho odd padded", **ortho, "pad": 5, "src": "fp32", "dst": "bf16",
         "shapes": "1x1000x777 3x333x2049 1x1x515 1x515x1 2x129x130"},
        # one layer's experts
        {"name": "ortho 64 experts bf16", **ortho, "shapes": "64x256x1024", "src": "bf16", "dst": "bf16"},
        # one large square weight in fp32
        {"name": "ortho 1x2048x2048 fp32", **ortho, "shapes": "1x2048x2048", "src": "fp32", "dst": "fp32"},
        # a large layer's square and wide weights
        {"name": "ortho 4096 and 8192", **ortho, "shapes": "1x4096x4096 1x2048x8192", "src": "fp32",
         "dst": "bf16"},
        # one small weight's step
        {"name": "muon 1x128x512 mixed", **muon, "shapes": "1x128x512", "layout": "bf16_mixed"},
        # the segmentation net's step, fp32
        {"name": "muon segnet fp32", **muon, "shapes": SEGNET, "layout": "fp32", "scale": "aspect",
         "lr": 1e-3, "wd": 0.05},
        # the mixed-precision list with its clip and loss scaler
        {"name": "muon 46M ragged mixed", **muon, "shapes": RAGGED, "layout": "bf16_mixed", "clip": 1.0,
         "scaler": True},
        # the 200M-parameter model's step
        {"name": "muon 200M layers mixed", **muon, "shapes": LAYERS, "layout": "bf16_mixed", "clip": 1.0},
    ]


def _dim(rng, lo=1, hi=4096):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["orthogonalize", "muon_step"])
    fp32 = rng.random() < 0.4
    budget = math.exp(rng.uniform(math.log(1e7), math.log(2e11 if fp32 else 6e11)))
    shapes = []
    for _ in range(rng.choice([1, 1, 2, 3, 5])):
        lo = rng.choice([1, 16, 64])
        # products of 32 bits keep their bound up to sides of about 2048
        r, c = _dim(rng, lo, 2048 if fp32 else 4096), _dim(rng, lo, 2048 if fp32 else 4096)
        cost = _flops(1, r, c)
        if cost > budget and shapes:
            continue
        most = max(1, min(64, int(budget / cost), int(5e7 / (r * c))))
        shapes.append("%dx%dx%d" % (rng.randint(1, most), r, c))
    case = {"op": op, "shapes": " ".join(shapes)}
    if op == "orthogonalize":
        case.update(src=rng.choice(["fp32", "bf16"]), dst="fp32" if fp32 else "bf16",
                    pad=rng.choice([0, 0, 1, 5, 8]))
    else:
        scale = rng.choice(["rms", "aspect", "none"])
        # the weights (rms 0.02) move by 4e-6 to 6e-5 a step, whichever factor is used
        # (an orthogonalised matrix has an rms of 1 / sqrt of its longer side)
        move = math.exp(rng.uniform(math.log(4e-6), math.log(6e-5)))
        lr = min(move * math.sqrt(max(r, c)) / _scale_of(scale, r, c) for _, r, c in _shapes(case))
        case.update(layout="fp32" if fp32 else "bf16_mixed", lr=lr, scale=scale,
                    momentum=rng.choice([0.9, 0.95]), nesterov=rng.random() < 0.7,
                    wd=rng.choice([0.0, 0.01, 0.1]), clip=rng.choice([0.0, 1.0]),
                    scaler=rng.random() < 0.5)
    return case


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split()]


def _matrices(gen, count, rows, cols, rms):
    """What a momentum looks like: a few strong directions over noise."""
    rank = max(1, min(rows, cols, 256) // 8)
    kw = dict(generator=gen, device="cuda", dtype=torch.float32)
    left = torch.randn(count, rows, rank, **kw) / torch.arange(1, rank + 1, device="cuda")
    x = torch.bmm(left, torch.randn(count, rank, cols, **kw))
    x += 0.2 * torch.randn(count, rows, cols, **kw)
    return x.mul_(rms)


def _padded(x, pad):
    """`x` as a slice of a buffer whose rows are `pad` elements longer."""
    if not pad:
        return x
    buf = torch.zeros(*x.shape[:-1], x.shape[-1] + pad, dtype=x.dtype, device=x.device)
    buf[..., :x.shape[-1]] = x
    return buf[..., :x.shape[-1]]


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shapes = _shapes(case)
    if case["op"] == "orthogonalize":
        return {"src": [_padded(_matrices(gen, *s, 1e-3).to(DTYPES[case["src"]]), case["pad"])
                        for s in shapes]}
    mixed = case["layout"] == "bf16_mixed"
    dtype = torch.bfloat16 if mixed else torch.float32
    scale = 65536.0 if case["scaler"] else 1.0
    return {"param": [(0.02 * torch.randn(s, generator=gen, device="cuda")).to(dtype) for s in shapes],
            "grad": [_matrices(gen, *s, 1e-3 * scale).to(dtype) for s in shapes],
            "momentum": [_matrices(gen, *s, 5e-3) for s in shapes]}


def prepare(case, seed):
    st = {"case": dict(case), **_inputs(case, seed)}
    if case["op"] == "orthogonalize":
        st["dst"] = [_padded(torch.zeros(s, dtype=DTYPES[case["dst"]], device="cuda"), case["pad"])
                     for s in _shapes(case)]
        if own:
            st["plan"] = _library().Orthogonalizer(st["src"], st["dst"])
    elif own:
        sb = _library()
        opt = sb.Muon(st["param"], sb.MuonOptions(
            lr=case["lr"], momentum=case["momentum"], nesterov=case["nesterov"],
            weight_decay=case["wd"], scale=case["scale"]), grads=st["grad"], layout=case["layout"],
            max_grad_norm=case["clip"],
            loss_scaler=sb.LossScalerOptions(init_scale=65536.0, growth_interval=1 << 30) if case["scaler"] else None)
        st["opt"] = opt
        views = [opt.state(i, sb.STATE_M).view(m.shape) for i, m in enumerate(st["momentum"])]
        for view, m in zip(views, st["momentum"]):  # training that was under way
            view.copy_(m)
        st["momentum"] = views
        st["master"] = [opt.state(i, sb.STATE_MASTER).view(p.shape) for i, p in enumerate(st["param"])]
    else:
        # (copies: the fp32 layout's master weights are the parameters)
        st["master"] = [p.float() for p in st["param"]]
    return st


def _library():
    path = str(Path("soar.cpp_b200").resolve())
    if path not in sys.path:
        sys.path.insert(0, path)
    import soar_b200
    return soar_b200


def _scale_of(mode, rows, cols):
    if mode == "rms":
        return 0.2 * math.sqrt(max(rows, cols))
    return math.sqrt(max(1.0, rows / cols)) if mode == "aspect" else 1.0


def _newton_schulz(g):
    """The plain form, on a stack [count, rows, cols], in 32 bits (the norm's long sum in 64)."""
    a, b, c = NS
    x = g.float()
    norm = x.double().square().sum(dim=(1, 2), keepdim=True).sqrt()
    x = x / (norm + EPS).float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    for _ in range(STEPS):
        xx = x @ x.transpose(1, 2)
        x = a * x + (b * xx + c * (xx @ xx)) @ x
    return x.transpose(1, 2) if tall else x


def run(state):
    case = state["case"]
    if case["op"] == "orthogonalize":
        if own:
            state["plan"].run()
        else:
            for src, dst in zip(state["src"], state["dst"]):
                dst.copy_(_newton_schulz(src))
        return list(state["dst"])
    if own:
        state["opt"].step()
    else:
        _muon_plain(state, case)
    out = {"param": list(state["param"]), "momentum": list(state["momentum"])}
    if case["layout"] == "bf16_mixed":
        out["master"] = list(state["master"])
    return out


def _muon_plain(state, case):
    inv = 1.0 / 65536.0 if case["scaler"] else 1.0
    coef = torch.ones((), device="cuda")
    keep = torch.ones((), device="cuda", dtype=torch.bool)
    if case["clip"] or case["scaler"]:
        total = sum((g.float() * inv).double().square().sum() for g in state["grad"])
        norm = total.sqrt().float()
        if case["clip"]:
            coef = torch.where((norm > case["clip"]) & (norm > 1e-6), case["clip"] / norm, coef)
        if case["scaler"]:
            keep = torch.isfinite(total)
    for p, w, g, m in zip(state["param"], state["master"], state["grad"], state["momentum"]):
        d = g.float() * inv * coef
        new_m = case["momentum"] * m + d
        u = d + case["momentum"] * new_m if case["nesterov"] else new_m
        s = case["lr"] * _scale_of(case["scale"], p.shape[1], p.shape[2])
        new_w = w - case["lr"] * case["wd"] * w - s * _newton_schulz(u)
        m.copy_(torch.where(keep, new_m, m))
        w.copy_(torch.where(keep, new_w, w))
        p.copy_(w)


def _flops(count, rows, cols):
    """The products X X^T and A A are symmetric: half of each is enough."""
    m, n = min(rows, cols), max(rows, cols)
    return count * STEPS * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)


def work(case):
    shapes = _shapes(case)
    values = sum(c * r * k for c, r, k in shapes)
    if case["op"] == "orthogonalize":
        size = {"fp32": 4, "bf16": 2}
        per = size[case["src"]] + size[case["dst"]]
    else:
        # gradient and weights in, momentum in and out, weights out (mixed: bf16 too)
        per = 2 + 8 + 8 + 2 if case["layout"] == "bf16_mixed" else 4 + 8 + 8
    return {"bytes": per * values, "flops": sum(_flops(*s) for s in shapes)}


def _polar64(g):
    """The operator's definition in 64 bits, matrix by matrix: X <- X (a I + b X^T X + c (X^T X)^2)
    on the columns' side, or the same on the rows' side where there are fewer rows."""
    a, b, c = NS
    out = torch.empty(g.shape, dtype=torch.float64, device=g.device)
    for i in range(g.shape[0]):
        x = g[i].double()
        x = x / (torch.linalg.vector_norm(x) + EPS)
        eye = torch.eye(min(x.shape), dtype=torch.float64, device=x.device)
        for _ in range(STEPS):
            if x.shape[0] < x.shape[1]:
                q = torch.mm(x, x.t())
                x = torch.mm(torch.addmm(b * q, q, q, alpha=c) + a * eye, x)
            else:
                q = torch.mm(x.t(), x)
                x = torch.mm(x, torch.addmm(b * q, q, q, alpha=c) + a * eye)
        out[i] = x
    return out


def exact(case, seed):
    if sum(_flops(*s) for s in _shapes(case)) > 5e13:
        return None
    data = _inputs(case, seed)
    if case["op"] == "orthogonalize":
        return [_polar64(x) for x in data["src"]]
    inv = 2.0 ** -16 if case["scaler"] else 1.0
    grads = [g.double() * inv for g in data["grad"]]
    factor = 1.0
    if case["clip"]:
        norm = math.sqrt(sum(float(torch.linalg.vector_norm(g)) ** 2 for g in grads))
        factor = min(1.0, case["clip"] / norm)
    out = {"param": [], "momentum": [], "master": []}
    for w, g, m in zip(data["param"], grads, data["momentum"]):
        m = torch.add(factor * g, m.double(), alpha=case["momentum"])
        u = torch.add(factor * g, m, alpha=case["momentum"]) if case["nesterov"] else m
        step = case["lr"] * _scale_of(case["scale"], *w.shape[1:])
        w = torch.add(w.double() * (1.0 - case["lr"] * case["wd"]), _polar64(u), alpha=-step)
        out["param"].append(w)
        out["momentum"].append(m)
        out["master"].append(w)
    if case["layout"] != "bf16_mixed":
        del out["master"]
    return out
