"""Group norm where its sizes are far apart: many samples of few places and wide groups."""
import pytest
import torch

from test_group_norm_hip import TYPES, _check, _inputs, _plan, _reference, _run


def test_workspace_of_many_samples():
    """Groups too wide to be held: what the gradients of weight and bias are added from is a fraction of x, not a row a sample."""
    from maloq_amd import _lib
    lib = _lib.load()
    for code, size in ((0, 4), (1, 2), (2, 2)):
        for n, p, c, groups in ((100000, 1, 8192, 1), (1000000, 1, 5000, 1), (30000, 4, 8192, 1), (100000, 2, 9000, 2), (5000, 3, 63000, 7), (3000, 40, 9000, 2), (3000, 9, 9000, 2)):
            for back in (0, 1):
                got = 4 * lib.maloq_group_norm_workspace_floats(code, n, p, c, groups, back)
                assert 0 <= got <= n * p * c * size / 4 + 2 ** 24, (n, p, c, groups, back)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,p,c,groups", [(5000, 1, 9000, 2), (3000, 2, 4504, 1), (700, 3, 20000, 1), (2053, 1, 4100, 1)])
def test_many_samples_of_wide_groups(n, p, c, groups, dt, device):
    """Workgroups that add the columns of several samples: sums of as many terms as there are places, in two levels."""
    plan = _plan(dt, n, p, c, groups, True)
    assert plan[0] == 0 and plan[6] < n * plan[4]
    x, w, b, g = (t.to(device) for t in _inputs(n, p, c, dt, seed=n))
    got = _run(x, w, b, g, groups, "silu")
    for t, (name, (value, bound)) in zip(got, _reference(x, w, b, g, groups, "silu", dt, 100).items()):
        _check(t, value, bound, name)
    assert all(torch.equal(a, e) for a, e in zip(_run(x, w, b, g, groups, "silu"), got))
