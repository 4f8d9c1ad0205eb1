"""Linear layers over empty contractions (maloq_amd.dense): act(bias) + residual, and gradients that are zero or the
bias's own; the few-rows kernel, tiles, and rows that need tiles of 128."""
import pytest
import torch

from test_dense_hip import ACTS, E32, HALVES, TINY, _act, _check, _slope, _u

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", HALVES + [torch.float32])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n", [(1, 1), (5, 24), (40, 24), (70, 133), (300, 260)])
def test_no_inner(m, n, act, dt, device):
    from maloq_amd.dense import linear_act
    gen = torch.Generator().manual_seed(m)
    make = lambda *s: torch.randn(*s, generator=gen).to(dt).to(device)
    x, w = (torch.empty(s, 0, device=device, dtype=dt, requires_grad=True) for s in (m, n))
    b, r, g = make(n).requires_grad_(), make(m, n), make(m, n)
    y = linear_act(x, w, b, act=act, residual=r)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g)
    assert gx.shape == (m, 0) and gw.shape == (n, 0)
    z, r64, g64 = b.detach().double().expand(m, n), r.double(), g.double()
    pre = _act(z, act)
    own = 2.0 ** -20 if dt != torch.float32 else 8 * E32  # an activation's error, of 16 bits and of fp32
    _check(y, pre + r64, own * (1 + z.abs()) * pre.abs() + 2 * E32 * (pre + r64).abs() + own * (dt == torch.float32), "y")
    dz = g64 * _slope(z, act)
    ez = own * (1 + z.abs()) * g64.abs() if act in ("silu", "gelu") else 0 * g64  # (the argument is the bias: stored as it is)
    _check(gb, dz.sum(0), ez.sum(0) + (m + 8) * E32 * dz.abs().sum(0), "db")
    assert torch.equal(linear_act(x, w, act=act), torch.zeros_like(y))


@pytest.mark.parametrize("out", HALVES + [torch.float32])
@pytest.mark.parametrize("m,n", [(5, 24), (70, 133)])
def test_no_inner_in_eight_bits(m, n, out, device):
    from maloq_amd.dense import linear_quantized
    q, p = (torch.empty(s, 0, device=device, dtype=torch.float8_e4m3fn) for s in (m, n))
    s, t = (torch.ones(c, device=device) for c in (m, n))
    b = torch.randn(n, device=device).to(out)
    assert torch.equal(linear_quantized(q, s, p, t, b, act="relu", dtype=out), torch.relu(b).expand(m, n))


@pytest.mark.parametrize("dt", HALVES + [torch.float32])
def test_no_rows_no_outer(dt, device):
    """No rows: gradients of weights and bias are zero.  No outputs: the gradient of x is zero."""
    from maloq_amd.dense import linear_act
    for m, k, n in ((0, 16, 24), (0, 9, 200), (5, 16, 0), (100, 200, 0)):
        x, w, b = (torch.randn(*s, device=device).to(dt).requires_grad_() for s in ((m, k), (n, k), (n,)))
        y = linear_act(x, w, b, act="silu")
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
        assert y.shape == (m, n) and gx.shape == (m, k) and gw.shape == (n, k) and gb.shape == (n,)
        assert not gx.any() and not gw.any() and not gb.any()
