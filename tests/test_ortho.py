"""soar_ortho_* / Orthogonalizer: the refusals (no GPU), and the results on the
GPU against the definition in 64 bits at the sizes, types, strides and values
where the kernels' tiles, splits and scales could go wrong."""
import ctypes

import pytest
import torch

import soar_b200 as sb
from matrix_helpers import matrices, ns64, rel, tolerance
from soar_b200 import optim

gpu = pytest.mark.gpu


# ------------------------------------------------------------ refusals (CPU) --

def _create(descs, **over):
    lib = sb.lib()
    o = optim.OrthoOpts()
    lib.soar_ortho_default_opts(ctypes.byref(o))
    for k, v in over.items():
        setattr(o, k, v)
    arr = (optim.MatrixDesc * max(1, len(descs)))(*descs)
    out = ctypes.c_void_p()
    rc = lib.soar_ortho_create(arr, len(descs), ctypes.byref(o), ctypes.byref(out))
    return rc, lib.soar_last_error().decode()


def _desc(src=4096, dst=8192, count=1, rows=4, cols=8, src_row=8, src_mat=32, dst_row=8, dst_mat=32):
    return optim.MatrixDesc(src, dst, count, rows, cols, src_row, src_mat, dst_row, dst_mat)


@pytest.mark.parametrize("desc,over,word", [
    (_desc(src=None), {}, "null"),
    (_desc(dst=None), {}, "null"),
    (_desc(src=4098), {}, "aligned"),
    (_desc(dst=8193), {}, "aligned"),
    (_desc(src_row=7), {}, "overlap"),
    (_desc(dst_row=7), {}, "overlap"),
    (_desc(count=3, dst_mat=31), {}, "overlap"),
    (_desc(rows=1, count=3, dst_mat=7), {}, "overlap"),
    (_desc(rows=(1 << 20) + 1), {}, "1048576"),
    (_desc(cols=(1 << 20) + 1, src_row=1 << 21, dst_row=1 << 21), {}, "1048576"),
    (_desc(count=1 << 40), {}, "2^38"),
    (_desc(rows=0, count=1 << 40), {}, "2^31"),
    (_desc(src_mat=1 << 41), {}, "stride"),
    (_desc(dst=4096), {}, "in place"),                      # fp32 into bf16
    (_desc(dst=4096, dst_row=9), {"dst_type": 0}, "in place"),
    (_desc(), {"steps": 0}, "steps"),
    (_desc(), {"steps": 17}, "steps"),
    (_desc(), {"eps": -1.0}, "eps"),
    (_desc(), {"eps": float("nan")}, "eps"),
    (_desc(), {"src_type": 2}, "type"),
    (_desc(), {"dst_type": -1}, "type"),
])
def test_refusals(desc, over, word):
    rc, why = _create([desc], **over)
    assert rc == -1 and word in why, why


def test_refuses_destinations_taken_and_strides_that_wrap():
    rc, why = _create([_desc(), _desc(src=1 << 20)])
    assert rc == -1 and "same destination" in why, why
    # (count - 1) x stride is past 64 bits
    rc, why = _create([_desc(count=1 << 26, dst_mat=1 << 40)])
    assert rc == -1 and "2^44" in why, why
    rc, why = _create([_desc(count=1 << 26, src_mat=1 << 40)])
    assert rc == -1 and "2^44" in why, why


def test_null_arguments():
    lib = sb.lib()
    assert lib.soar_ortho_create(None, 1, None, None) == -1
    assert lib.soar_ortho_run(None, None) == -1
    assert lib.soar_ortho_error(None, None) == -1
    assert lib.soar_ortho_destroy(None) == -1


def test_python_refusals():
    a = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        sb.Orthogonalizer([a], [a.clone()])
    with pytest.raises(ValueError, match="one destination"):
        sb.Orthogonalizer([a], [])
    with pytest.raises(ValueError, match="more than one type"):
        sb.Orthogonalizer([a, a.bfloat16()], [a, a])
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        sb.Orthogonalizer([a.half()], [a])
    with pytest.raises(ValueError, match="coefficients"):
        sb.Orthogonalizer([a], [a], sb.OrthogonalizeOptions(steps=3, coefficients=((1, 2, 3),) * 2))
    with pytest.raises(ValueError, match="steps"):
        sb.Orthogonalizer([a], [a], sb.OrthogonalizeOptions(steps=17))


# ------------------------------------------------------------ results (GPU) ---

def _run(srcs, dst_dtype, options=None, pad=0):
    dev = [s.cuda() for s in srcs]
    if pad:
        dev = [torch.nn.functional.pad(s, (pad, 2 * pad))[..., pad:pad + s.shape[-1]] for s in dev]
        dsts = [torch.full((*s.shape[:-1], s.shape[-1] + 3 * pad), 7.0, dtype=dst_dtype,
                           device="cuda")[..., pad:pad + s.shape[-1]] for s in srcs]
    else:
        dsts = [torch.full(s.shape, 7.0, dtype=dst_dtype, device="cuda") for s in srcs]
    plan = sb.Orthogonalizer(dev, dsts, options)
    plan.run()
    torch.cuda.synchronize()
    assert plan.error() == 0
    return dsts, plan


SHAPES = [(1, 1), (1, 2), (2, 1), (7, 5), (1, 515), (515, 1), (16, 16), (17, 33), (63, 65), (64, 64),
          (65, 63), (100, 128), (128, 128), (129, 127), (128, 700), (700, 130), (255, 257), (256, 256),
          (257, 300), (384, 384), (513, 1000), (1000, 640), (1030, 1025)]


@gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
@pytest.mark.parametrize("src,dst", [("float32", "float32"), ("float32", "bfloat16"),
                                     ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
def test_matches_definition(cuda, shape, src, dst):
    src, dst = getattr(torch, src), getattr(torch, dst)
    for kind in ("spectrum", "noise"):
        g = matrices((1, *shape), 5 + shape[0], kind).to(src)[0]
        want = ns64(g.cuda())
        (got,), _ = _run([g], dst)
        assert rel(got, want) <= tolerance(g.cuda(), want, dst), (kind, rel(got, want))


@gpu
@pytest.mark.parametrize("dst", [torch.float32, torch.bfloat16])
def test_list_of_stacks_padded(cuda, dst):
    """Stacks of many shapes in one call, rows inside larger buffers: the
    elements around them stay, and every matrix is as if it were alone."""
    shapes = [(3, 40, 77), (1, 200, 130), (5, 129, 33), (2, 64, 300), (1, 1, 9), (4, 300, 280), (7, 8, 8)]
    gs = [matrices(s, 40 + i) for i, s in enumerate(shapes)]
    got, plan = _run(gs, dst, pad=3)
    for g, d in zip(gs, got):
        for i in range(g.shape[0]):
            want = ns64(g[i].cuda())
            assert rel(d[i], want) <= tolerance(g[i].cuda(), want, dst)
        rows = g.shape[0] * g.shape[1]
        buf = d._base.reshape(rows, -1) if d._base is not None else d
        assert bool((buf[:, :3] == 7).all()) and bool((buf[:, 3 + g.shape[2]:] == 7).all())


@gpu
@pytest.mark.parametrize("shapes", [[(1, 130, 1152)], [(1, 130, 1153)], [(2, 4100, 100)], [(1, 1, 20000)],
                                    [(2, 256, 1300), (80, 90, 1400)], [(3, 240, 5001), (1, 33, 64), (1, 300, 310)]],
                         ids=lambda s: "+".join("x".join(map(str, v)) for v in s))
def test_long_matrices_of_few_rows(cuda, shapes):
    """At most 256 rows: alone, where the longest columns are dealt to all SMs,
    and in lists long enough for a pair of CTAs per matrix."""
    gs = [matrices(s, 60 + i) for i, s in enumerate(shapes)]
    got, _ = _run(gs, torch.bfloat16)
    for g, d in zip(gs, got):
        want = ns64(g.cuda())
        assert rel(d, want) <= tolerance(g.cuda(), want, torch.bfloat16)


@gpu
def test_values(cuda):
    """Zeros give zeros; one inf or NaN makes its matrix NaN and no other; very
    small, very large and one-element matrices come out as the definition says."""
    g = matrices((8, 96, 160), 3)
    g[0] = 0
    g[1, 5, 6] = float("inf")
    g[2, 95, 159] = float("nan")
    g[3] *= 1e-30          # (values near 1e-33: still normal numbers)
    g[4] *= 1e18
    g[5] = 0
    g[5, 17, 3] = 2.5      # all of the norm in one element
    g[6] = 1.0             # rank one
    for dst in (torch.float32, torch.bfloat16):
        (got,), _ = _run([g], dst)
        assert bool((got[0] == 0).all())
        assert bool(got[1].isnan().all()) and bool(got[2].isnan().all())
        for i in (4, 5, 6, 7):
            want = ns64(g[i].cuda())
            assert rel(got[i], want) <= tolerance(g[i].cuda(), want, dst), i
        # eps (1e-7) outweighs the norm of g[3]: the result is g / eps through the iteration
        want = ns64(g[3].cuda())
        assert float((got[3].double() - want).abs().max()) <= 1e-4 * float(want.abs().max()) + 1e-10


@gpu
def test_coefficients_per_step(cuda):
    """Another number of steps, each with its own coefficients."""
    coef = ((4.0, -6.0, 2.5), (3.0, -3.2, 1.2), (1.875, -1.25, 0.375))
    g = matrices((2, 150, 90), 12)
    for dst in (torch.float32, torch.bfloat16):
        (got,), _ = _run([g], dst, sb.OrthogonalizeOptions(steps=3, coefficients=coef))
        want = ns64(g.cuda(), steps=3, coef=coef)
        assert rel(got, want) <= tolerance(g.cuda(), want, dst, steps=3, coef=coef)
    (got,), _ = _run([g], torch.float32, sb.OrthogonalizeOptions(steps=1))
    want = ns64(g.cuda(), steps=1)
    assert rel(got, want) <= tolerance(g.cuda(), want, torch.float32, steps=1)


@gpu
def test_in_place_repeat_stream_graph(cuda):
    """A run in place; the same bits from every run, on another stream, and from
    a captured and replayed one after its input changed."""
    g = matrices((3, 130, 260), 9)
    x = g.cuda()
    sb_in_place = sb.Orthogonalizer([x], [x])
    sb_in_place.run()
    (want,), plan = _run([g], torch.float32)
    assert torch.equal(x, want)
    src, dst = plan.srcs[0], plan.dsts[0]
    first = dst.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    dst.zero_()
    torch.cuda.synchronize()
    plan.run(stream)
    stream.synchronize()
    assert torch.equal(dst, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run()
    src.copy_(matrices((3, 130, 260), 10))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    (other,), _ = _run([matrices((3, 130, 260), 10)], torch.float32)
    assert torch.equal(dst, other) and not torch.equal(dst, first)


@gpu
@pytest.mark.parametrize("shape", [(3, 130, 260), (5, 100, 64), (1, 600, 520)], ids=str)
def test_in_place_runs_back_to_back(cuda, shape):
    """Each run in place takes the last one's result: as two runs between buffers."""
    for dt in (torch.float32, torch.bfloat16):
        x, y = matrices(shape, 11).to(dt).cuda(), torch.empty(shape, dtype=dt, device="cuda")
        there, back = sb.Orthogonalizer([x], [y]), sb.Orthogonalizer([y], [x])
        z = x.clone()
        in_place = sb.Orthogonalizer([z], [z])
        for _ in range(4):
            in_place.run()
            in_place.run()
            there.run()
            back.run()
        torch.cuda.synchronize()
        assert torch.equal(z, x)


@gpu
def test_two_plans_on_two_streams(cuda):
    """Runs of two plans at once, many tiles each: neither waits for the other."""
    gs = [matrices((24, 256, 384), 20), matrices((2, 900, 1100), 21)]
    alone = [_run([g], torch.bfloat16)[0][0].clone() for g in gs]
    made = [_run([g], torch.bfloat16) for g in gs]
    streams = [torch.cuda.Stream() for _ in gs]
    torch.cuda.synchronize()
    for _ in range(6):
        for (dsts, plan), s in zip(made, streams):
            plan.run(s)
    torch.cuda.synchronize()
    for ((dst,), plan), want in zip(made, alone):
        assert plan.error() == 0 and torch.equal(dst, want)


@gpu
@pytest.mark.parametrize("src", [torch.float32, torch.bfloat16])
def test_many_runs_of_ragged_lists(cuda, src):
    """Runs back to back, by turns, of lists of many matrices of a few tiles each:
    every pair of CTAs goes through hundreds of tiles of changing shape and chunk
    counts, some without rows for its second CTA, and through several matrices
    of at most 256 rows. No wait gives up, and every run leaves the same bits."""
    shapes = [(24, 128, 131), (24, 130, 192), (24, 250, 257), (24, 320, 320), (24, 300, 400), (24, 512, 250),
              (24, 400, 400), (24, 640, 300), (16, 480, 480), (16, 385, 510)]
    gen = torch.Generator(device="cuda").manual_seed(5)
    lists = [[torch.randn(s, generator=gen, device="cuda").to(src) for s in shapes] for _ in range(2)]
    dsts = [[torch.empty_like(x) for x in xs] for xs in lists]
    plans = [sb.Orthogonalizer(xs, ys) for xs, ys in zip(lists, dsts)]
    first = []
    for plan, ys in zip(plans, dsts):
        plan.run()
        first.append([y.clone() for y in ys])
    for _ in range(10):
        for _ in range(30):
            for plan in plans:
                plan.run()
        torch.cuda.synchronize()
        for plan, ys, want in zip(plans, dsts, first):
            assert plan.error() == 0
            assert all(torch.equal(y, w) for y, w in zip(ys, want))


@gpu
def test_empty(cuda):
    plan = sb.Orthogonalizer([], [])
    plan.run()
    e = torch.zeros(3, 0, 5, device="cuda")
    sb.Orthogonalizer([e], [e.clone()]).run()
    torch.cuda.synchronize()


@gpu
def test_permuted_strides(cuda):
    """A stack whose matrices are interleaved row by row, and refused strides."""
    base = matrices((40, 3, 64), 2).cuda()          # [rows, count, cols]
    src = base.permute(1, 0, 2)
    out = torch.zeros_like(base)
    sb.Orthogonalizer([src], [out.permute(1, 0, 2)]).run()
    for i in range(3):
        want = ns64(src[i])
        assert rel(out[:, i], want) <= tolerance(src[i], want, torch.float32)
    with pytest.raises(ValueError, match="contiguous"):
        sb.Orthogonalizer([base[0].t()], [base[0].t().clone()])
    flat = torch.zeros(1, 64, device="cuda").expand(5, 64)
    with pytest.raises(sb.SoarError, match="overlap"):
        sb.Orthogonalizer([torch.zeros(5, 64, device="cuda")], [flat])
