"""Lists that no device holds are refused before the host plans them."""
import resource

import pytest

import soar_b200 as sb
from soar_b200 import optim
from test_ortho import _create

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("desc", [
    optim.MatrixDesc(1 << 20, 1 << 40, (1 << 31) - 1, 1, 1, 1, 1, 1, 1),
    optim.MatrixDesc(1 << 20, 1 << 40, 1 << 18, 1 << 10, 1 << 10, 1 << 10, 1 << 20, 1 << 10, 1 << 20)])
@pytest.mark.parametrize("dst", [0, 1])
def test_refuses_more_than_the_device_holds(cuda, desc, dst):
    sb.Orthogonalizer([], []).close()  # (what a first call allocates is no part of it)
    before = resource.getrusage(resource.RUSAGE_SELF).ru_maxrss
    rc, why = _create([desc], dst_type=dst)
    assert rc == -1 and "memory" in why, why
    assert resource.getrusage(resource.RUSAGE_SELF).ru_maxrss - before < 1 << 20  # KB
