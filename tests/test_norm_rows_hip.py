"""The residual norm's backward (maloq_amd.norm) with more rows than it has workgroups, at every number of threads a
row: the second and later rows of a workgroup, and dw carried over them.  Bounds as in test_norm_hip."""
import pytest
import torch

from test_norm_hip import E32, TYPES, _check, _inputs, _reference, _u

pytestmark = pytest.mark.gpu


# sixteen threads a row (8193 rows are more than 512 workgroups have), one wave, four, eight, sixteen
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,n", [(8300, 128), (8195, 40), (2100, 500), (2085, 1000), (1100, 2040), (1100, 4096), (1037, 8192),
                                    (1100, 12345), (1100, 16384)])
@pytest.mark.parametrize("residual", [True, False])
def test_gradients_of_many_rows(rows, n, residual, dt, device):
    from maloq_amd.norm import rms_norm
    x, r, w, g, gh = _inputs(rows, n, dt, seed=rows + n)
    lx, lw = (t.to(device).requires_grad_() for t in (x, w))
    if residual:
        lr = r.to(device).requires_grad_()
        y, h = rms_norm(lx, lw, 1e-6, residual=lr)
        gx, gr, gw = torch.autograd.grad((y, h), (lx, lr, lw), (g.to(device), gh.to(device)))
        assert torch.equal(gx, gr)
    else:
        y = rms_norm(lx, lw, 1e-6)
        gx, gw = torch.autograd.grad(y, (lx, lw), g.to(device))
    # (the reference on the GPU, compared there)
    x, r, w, g, gh = (t.to(device) for t in (x, r, w, g, gh))
    h64, rstd, y64 = _reference(x, r if residual else None, w, 1e-6)
    g64, u64 = g.double(), g.double() * w.double()
    dot, dot_abs = (u64 * h64).mean(-1, keepdim=True), (u64 * h64).abs().mean(-1, keepdim=True)
    f = rstd ** 2 * dot
    dx = rstd * (u64 - h64 * f) + (gh.double() if residual else 0)
    e = _u(dt) + 48 * E32
    bx = rstd * (8 * E32 * u64.abs() + h64.abs() * (e * f.abs() + rstd ** 2 * dot_abs * e * 2)) \
        + (48 + 8) * E32 * rstd * (u64.abs() + (h64 * f).abs()) + 2 * E32 * dx.abs()
    terms = g64 * h64 * rstd
    _check(y, y64.cpu(), (48 * E32 * y64.abs()).cpu(), dt, "y")
    _check(gx, dx.cpu(), bx.cpu(), dt, "dx")
    _check(gw, terms.sum(0).cpu(), (terms.abs().sum(0) * (e + (rows + 8) * E32)).cpu(), dt, "dw")
