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


def _same_way(dt, n, few, p, c, groups, backward):
    """Whether so many samples take the kernels, and so the order of sums, that few do."""
    return _plan(dt, n, p, c, groups, backward)[:6] + _plan(dt, n, p, c, groups, backward)[7:] == _plan(dt, few, p, c, groups, backward)[:6] + _plan(dt, few, p, c, groups, backward)[7:]


@pytest.mark.gpu
def test_more_samples_than_one_launch_forward(device):
    """2^29 rows of 33 values by eight threads each, of one row of memory: all as in a launch of few."""
    from maloq_amd.norm import group_norm
    n, few, c = (1 << 29) + 100, 100000, 33
    assert _same_way(torch.bfloat16, n, few, 1, c, 1, False) and _plan(torch.bfloat16, n, 1, c, 1, False)[0]
    x = torch.randn(1, c, generator=torch.Generator().manual_seed(0)).bfloat16().to(device)
    y, one = group_norm(x.expand(n, c), 1, act="silu"), group_norm(x.expand(few, c), 1, act="silu")[:1]
    for first in range(0, n, 1 << 26):
        assert bool((y[first:first + (1 << 26)] == one).all()), first


@pytest.mark.gpu
def test_more_samples_than_one_launch_step(device):
    """Wide groups, ten tiles of 256 threads a sample: dx in two launches, dw and db as one sample's times their number (but for
    the fp32 sums: a workgroup adds the columns of n / 204 samples, one after the other)."""
    n, few, c, dt = 1700000, 20000, 5000, torch.bfloat16
    plan = _plan(dt, n, 1, c, 1, True)
    assert _same_way(dt, n, few, 1, c, 1, False) and _same_way(dt, n, few, 1, c, 1, True) and plan[0] == 0 and n * plan[3] * 256 > 2 ** 32
    x, w, b, g = (t.to(device) for t in _inputs(1, 1, c, dt, seed=1))
    y, dx, dw, db = _run(x.expand(n, 1, c), w, b, g.expand(n, 1, c), 1, "silu")
    one = _run(x.expand(few, 1, c), w, b, g.expand(few, 1, c), 1, "silu")
    for t, e in ((y, one[0][:1]), (dx, one[1][:1])):
        for first in range(0, n, 200000):
            assert bool((t[first:first + 200000] == e).all()), first
    ref = _reference(x, w, b, g, 1, "silu", dt, 100)
    for t, name in ((dw, "dw"), (db, "db")):
        value, bound = ref[name]
        _check(t, n * value, n * (bound + (100 + n / plan[6]) * 2.0 ** -24 * value.abs()), name)
