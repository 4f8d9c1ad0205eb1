"""Linear layers (maloq_amd.dense) where an activation's argument passes the range of the tensors' type: fp32 sums
beyond +-65504 are stored for the backward as infinities of fp16.  Bounds as in test_dense_hip; beyond +-64 a slope
is 0 or 1 to within 2^-24, whatever the argument's own error."""
import pytest
import torch

from test_dense_hip import E32, HALVES, TINY, _act, _inputs, _slope, _u

pytestmark = pytest.mark.gpu


def _check(got, ref, bound, what):
    want = ref.to(got.dtype)
    far = want.isinf()  # (beyond the type)
    assert torch.equal(got[far], want[far]), what
    err, lim = (got.double() - ref)[~far].abs(), (bound + _u(got.dtype) * ref.abs() + TINY[got.dtype])[~far]
    assert bool((err <= lim * (1 + 1e-6)).all()), (what, (err / lim.clamp_min(1e-300)).max().item())


# a few rows; tiles of 64 and 128 rows; a contraction in parts; rows that are padded
@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("m,k,n", [(3, 40, 24), (40, 64, 130), (300, 96, 200), (100, 4096, 64), (300, 33, 40)])
def test_arguments_beyond_fp16(m, k, n, act, device):
    from maloq_amd.dense import linear_act
    dt = torch.float16
    x, w, b, _, g = (t.to(device) for t in _inputs(m, k, n, dt, seed=m + k))
    x[0, 0], x[m - 1, k - 1] = 280, -280
    w[0, 0], w[1, 0], w[n - 1, k - 1] = -250, 250, 250  # arguments about -70000, 70000, -70000
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = linear_act(*leaves, act=act)
    gx, gw, gb = torch.autograd.grad(y, leaves, g)
    x, w, b, g = (t.double() for t in (x, w, b, g))
    z = x @ w.T + b
    assert z.min() < -65520 and z.max() > 65520
    pre = _act(z, act)
    bz = (k + 8) * E32 * (x.abs() @ w.abs().T + b.abs())
    _check(y, pre, 1.13 * bz + 2.0 ** -20 * (1 + z.abs()) * pre.abs() + 2 * E32 * pre.abs(), "y")
    slope = _slope(z, act)
    dz = g * slope
    near = (z.abs() <= 64).double()
    if act == "relu":
        ez = g.abs() * (z.abs() <= bz + TINY[dt])
    else:
        ez = g.abs() * (near * (0.8 * (_u(dt) * z.abs() + bz + TINY[dt]) + 2.0 ** -20 * (1 + z.abs())) + E32)
    er = ez + _u(dt) * dz.abs() + TINY[dt]
    _check(gx, dz @ w, er @ w.abs() + (n + 8) * E32 * (dz.abs() @ w.abs()), "dx")
    _check(gw, dz.T @ x, er.T @ x.abs() + (m + 8) * E32 * (dz.abs().T @ x.abs()), "dw")
    _check(gb, dz.sum(0), ez.sum(0) + (m + 8) * E32 * dz.abs().sum(0), "db")


@pytest.mark.parametrize("dt", HALVES + [torch.float32])
@pytest.mark.parametrize("act,code", [("relu", 1), ("silu", 2), ("gelu", 3)])
def test_slopes_of_infinite_arguments(act, code, dt, device):
    """0 and 1, their limits; NaN stays.  (One row: its db is the slopes.)"""
    from maloq_amd import ops
    z = torch.tensor([[-float("inf"), float("inf"), float("nan"), -1e4, 1e4]], device=device).to(dt)
    x, w = torch.zeros(1, 8, device=device, dtype=dt), torch.zeros(5, 8, device=device, dtype=dt)
    db = ops.linear_act_bwd(torch.ones_like(z), x, w, z, code, False, False, True)[2]
    assert db[2].isnan() and torch.equal(db[[0, 1, 3, 4]], torch.tensor([0, 1, 0, 1], device=device).to(dt))
