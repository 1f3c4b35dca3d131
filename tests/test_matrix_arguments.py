"""Tensors that the matrix operators' Python classes would read wrongly are refused: a layout,
type, order or device other than the kernels take."""
import pytest
import torch

import soar_b200 as sb

gpu = pytest.mark.gpu


@pytest.mark.parametrize("param,grad,layout,word", [
    (torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16), "fp32", "float32"),
    (torch.zeros(4, 8), torch.zeros(4, 8), "bf16_mixed", "bfloat16"),
    (torch.zeros(4, 8), torch.zeros(4, 8, dtype=torch.bfloat16), "fp32", "gradient 0"),
    (torch.zeros(4, 8), torch.zeros(8, 4), "fp32", "gradient 0"),
    (torch.zeros(4, 8), torch.zeros(8, 4).t(), "fp32", "not contiguous"),
    (torch.zeros(4, 8), torch.zeros(4, 16)[:, ::2], "fp32", "not contiguous"),
    (torch.zeros(4, 8), torch.zeros(1, 8).expand(4, 8), "fp32", "not contiguous"),
    (torch.zeros(4, 8), torch.zeros(4, 8), "fp16", "layout"),
    (torch.zeros(4, 8), torch.zeros(4, 8), "fp32", "CUDA"),
    (torch.zeros(4, 8), None, "fp32", "CUDA"),
])
def test_muon_refuses(param, grad, layout, word):
    with pytest.raises(ValueError, match=word):
        sb.Muon([param], grads=[grad], layout=layout)


def test_muon_takes_iterators(monkeypatch):
    """As model.parameters() is one: every parameter reaches the library."""
    ps = [torch.nn.Parameter(torch.zeros(4, 8)) for _ in range(3)]
    seen = []
    monkeypatch.setattr(sb.Muon, "_check_tensors", staticmethod(lambda *a: None))
    monkeypatch.setattr(sb.Muon, "_create", lambda self, params, grads, *a: seen.append((
        [q for p in params for q in (p.params if isinstance(p, sb.ParamGroup) else [p])], list(grads))))
    sb.Muon(iter(ps))
    sb.Muon([sb.ParamGroup(iter(ps[:2]), 0.1), ps[2]], grads=iter([None] * 3))
    for params, grads in seen:
        assert all(a is b for a, b in zip(params, ps)) and len(params) == len(grads) == 3


def test_muon_refuses_a_grad_attribute_of_another_order():
    p = torch.nn.Parameter(torch.zeros(4, 8))
    p.grad = torch.zeros(4, 8).as_strided((4, 8), (1, 4))
    with pytest.raises(ValueError, match="not contiguous"):
        sb.Muon([p])
    with pytest.raises(ValueError, match="one gradient"):
        sb.Muon([p], grads=[])


@gpu
def test_on_the_device(cuda):
    w, g = torch.zeros(4, 8, device="cuda"), torch.zeros(4, 8, device="cuda")
    opt = sb.Muon([w], grads=[g])
    for bad in (torch.zeros(8, 4, device="cuda").t(), g.bfloat16(), torch.zeros(4, 8)):
        with pytest.raises(ValueError):
            opt.add_grads([bad])
    with pytest.raises(ValueError, match="1 gradient"):
        opt.add_grads([])
    assert opt.add_grads([g.clone()]) == 1
    with pytest.raises(ValueError, match="device"):
        sb.Muon([w], grads=[g], device=1)
    with pytest.raises(ValueError, match="device"):
        sb.Orthogonalizer([w], [g], device=1)
    with pytest.raises(ValueError, match="CUDA"):
        sb.Muon([w], grads=[torch.zeros(4, 8)])
    flat = torch.zeros(100, device="cuda")
    sb.Muon([w], grads=[flat[10:42]]).step()
    torch.cuda.synchronize()


@gpu
def test_added_gradients_on_another_stream(cuda):
    """A set that was just added, used at once by a stream that waits for no other."""
    from matrix_helpers import matrices
    ws = [torch.zeros(64, 96, device="cuda") for _ in range(2)]
    gs = [matrices((64, 96), i).cuda() for i in range(6)]
    opts = sb.MuonOptions(momentum=0.0, nesterov=False)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i, g in enumerate(gs):
        a, b = (w.zero_() for w in ws)
        one = sb.Muon([a], opts, grads=[gs[0]])
        two = sb.Muon([b], opts, grads=[g])
        torch.cuda.synchronize()
        one.use_grads(one.add_grads([g]))
        one.step(stream)
        two.step(stream)
        stream.synchronize()
        assert torch.equal(a, b), i
