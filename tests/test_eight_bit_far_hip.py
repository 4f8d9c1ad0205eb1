"""Gradients whose offsets pass 2^32: kept rows read back and unpacked, and group norm's backward by both its ways."""
import pytest
import torch

from test_group_norm_bounds_hip import Way
from test_group_norm_hip import _inputs, _plan, _reference, _run
from test_group_norm_limits_hip import _same_way

pytestmark = pytest.mark.gpu

ROWS, WIDE = 70000, 65536  # 4.6e9 values
SOME = [0, 1, 32768, 65535, 65536, 65537, 69998, ROWS - 1]


def test_kept_argument_in_the_weights_gradient(device):
    """Eight rows of x are unit vectors and their gradients alone are not zero: each column of dw is one row of the activation's
    gradient, as a layer of these rows only gives it."""
    from maloq_amd.dense import linear_act
    gen = torch.Generator().manual_seed(0)
    w = torch.randn(WIDE, 8, generator=gen).bfloat16().to(device)
    x = torch.randn(ROWS, 8, generator=gen).bfloat16().to(device)
    x[SOME] = torch.eye(8, device=device, dtype=torch.bfloat16)
    g = torch.zeros(ROWS, WIDE, device=device, dtype=torch.bfloat16)
    g[SOME] = torch.randn(8, WIDE, generator=gen).bfloat16().to(device)

    def step(x, g):
        leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
        return torch.autograd.grad(linear_act(*leaves, act="silu", checkpoint=torch.int8), leaves, g)

    gx, gw = step(x, g)
    small = torch.cat([x[SOME], x[2:50]])  # (more than 16 rows: the same kernels)
    want = step(small, torch.cat([g[SOME], torch.zeros_like(g[:48])]))
    assert torch.equal(gw, want[1])
    assert bool((gx[SOME].float() - want[0][:8].float()).norm() <= 2.0 ** -7 * want[0][:8].float().norm())
    rest = torch.ones(ROWS, dtype=torch.bool, device=device)
    rest[SOME] = False
    assert not gx[rest].any()


@pytest.mark.parametrize("k", [WIDE, WIDE - 3])
def test_kept_rows_in_the_weights_gradient(k, device):
    """Wide rows and a narrow weight: with a gradient of one in a row, dw's row is x's as it was kept."""
    from maloq_amd.dense import linear_act, pack_rows, unpack_rows
    gen = torch.Generator().manual_seed(1)
    base = torch.randn(1, k, generator=gen).bfloat16().to(device)
    x = base.repeat(ROWS, 1)
    x[SOME] *= torch.arange(1, 9, device=device, dtype=torch.bfloat16)[:, None]
    w = torch.zeros(8, k, device=device, dtype=torch.bfloat16).requires_grad_()
    g = torch.zeros(ROWS, 8, device=device, dtype=torch.bfloat16)
    g[SOME, torch.arange(8, device=device)] = 1
    gw, = torch.autograd.grad(linear_act(x, w, checkpoint=torch.int8), w, g)
    assert torch.equal(gw, unpack_rows(*pack_rows(x[SOME]), torch.bfloat16))


def test_held_group_norm(device):
    """300000 samples of 16 x 1024 values, all one: as in a launch of few."""
    n, few, p, c, groups, dt = 300000, 3000, 16, 1024, 8, torch.bfloat16
    assert _same_way(dt, n, few, p, c, groups, False) and _same_way(dt, n, few, p, c, groups, True) and _plan(dt, n, p, c, groups, True)[0]
    x, w, b, g = (t.to(device) for t in _inputs(1, p, c, dt, seed=1))
    got = _run(x.expand(n, p, c), w, b, g.expand(n, p, c), groups, "silu")
    one = _run(x.expand(few, p, c), w, b, g.expand(few, p, c), groups, "silu")
    for t, e in zip(got[:2], one[:2]):
        for first in range(0, n, 50000):
            assert bool((t[first:first + 50000] == e[:1]).all()), first
    steps = Way(dt, n, p, c, groups, True).columns + 64  # (a workgroup adds n / 1024 samples' columns one after the other)
    ref = _reference(x, w, b, g, groups, "silu", dt, steps)
    for t, name in zip(got[2:], ("dw", "db")):
        value, bound = ref[name]
        assert bool(((t.double() - n * value).abs() <= 2.0 ** -8 * n * value.abs() + n * bound).all()), name


@pytest.mark.parametrize("groups", [1, 4000])
def test_group_norm_in_parts(groups, device):
    """Places that are all alike: dx is one place's, db and dw that times their number.  A thread adds up to 3400 of them one after
    the other: the fp32 sums are off by as many 2^-24 of their terms."""
    p, c, dt = 40000, 60000, torch.bfloat16
    assert _plan(dt, 2, p, c, groups, True)[0] == 0
    x, w, b, g = (t.to(device) for t in _inputs(1, 1, c, dt, seed=2))
    y, dx, dw, db = _run(x.expand(2, p, c), w, b, g.expand(2, p, c), groups, "silu")
    ways = [Way(dt, 2, p, c, groups, back) for back in (False, True)]
    ref = _reference(x, w, b, g, groups, "silu", dt, max(ways[0].mean, ways[1].sums, ways[1].columns))
    for t, name in ((y, "y"), (dx, "dx")):
        value, bound = (v[0, 0] for v in ref[name])
        for at in ((0, 0), (0, 31582), (0, p - 1), (1, 0), (1, 31582), (1, p - 1)):
            assert bool(((t[at].double() - value).abs() <= 2.0 ** -8 * value.abs() + bound).all()), (name, at)
    for t, name in ((dw, "dw"), (db, "db")):
        value, bound = ref[name]
        assert bool(((t.double() - 2 * p * value).abs() <= 2.0 ** -8 * 2 * p * value.abs() + 2 * p * bound).all()), name
