"""The error word of the matrix operators reports a run whose wait gave up; it is not that
run's reason to fail, nor a later one's."""
import pytest
import torch

import soar_b200 as sb
from soar_b200.optim import _DeviceArray

gpu = pytest.mark.gpu

ERROR = 56  # bytes from the control block's start (the loss scale) to its error word


def _error_word(opt):
    return torch.as_tensor(_DeviceArray(opt.loss_scale_ptr() + ERROR, 1, "<i4", owner=opt), device="cuda")


@gpu
def test_a_run_after_a_reported_one_is_whole(cuda):
    """With the word set beforehand, as a run whose wait gave up leaves it. Few tiles of great
    depth: other pairs of CTAs poll for milliseconds until their inputs are there."""
    shape = (300, 1 << 18)
    gen = torch.Generator(device="cuda").manual_seed(1)
    g = 1e-3 * torch.randn(shape, generator=gen, device="cuda")
    results = []
    for word in (0, 1):
        w = torch.zeros(shape, device="cuda")
        opt = sb.Muon([w], sb.MuonOptions(lr=1.0, scale="none"), grads=[g])
        _error_word(opt).fill_(word)
        torch.cuda.synchronize()
        assert opt.info().error == word
        opt.step()
        info = opt.info()
        assert info.error == word and info.step == 1
        results.append(w)
        opt.set_counters(info.step, 0, 1.0, 0)
        assert opt.info().error == 0
        opt.close()
    assert bool(results[0].any()) and torch.equal(results[0], results[1])
