"""The residual norm (maloq_amd.norm) and 8-bit rows against 64 bits.

Bounds, each value for itself: an output of type t is rounded once (u = eps(t) / 2 of the value; a
16-bit value below the normal numbers by at most half of the least); h = x + r is one fp32
addition; a row's fp32 sums are chains of at most 8 products, then 2 + 6 + 16 additions, and what
follows them is a handful of operations: 48 steps of 2^-24.  The backward starts from the rounded
h (u of each of its values) and sums dw over the rows.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
E32 = 2.0 ** -24
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
WIDTHS = [1, 7, 8, 96, 97, 128, 256, 264, 513, 1000, 1024, 2047, 2048, 4096, 5001, 8192, 12345, 16384]


def _u(dt):
    return torch.finfo(dt).eps / 2


def _inputs(rows, n, dt, seed=0, n_more=0):
    gen = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=gen).to(dt)
    x, r, g, gh = (make(rows, n) for _ in range(4))
    return x, 2 * r, (1 + 0.2 * torch.randn(n, generator=gen)).to(dt), g, gh


def _check(got, ref, bound, dt, what):
    err = (got.double().cpu() - ref).abs()
    lim = bound + _u(dt) * ref.abs() + TINY[dt]
    assert got.dtype == dt and bool((err <= lim * (1 + 1e-6)).all()), (what, (err / lim.clamp_min(1e-300)).max().item())


def _reference(x, r, w, eps):
    h = x.double() if r is None else x.double() + r.double()
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    return h, rstd, h * rstd * w.double()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("rows", [1, 19])
@pytest.mark.parametrize("residual", [True, False])
def test_forward_and_gradients(rows, n, residual, dt, device):
    from maloq_amd.norm import rms_norm
    x, r, w, g, gh = _inputs(rows, n, dt, seed=n)
    r = r if residual else None
    eps = 1e-5
    lx, lw = (t.to(device).requires_grad_() for t in (x, w))
    lr = r.to(device).requires_grad_() if residual else None
    out = rms_norm(lx, lw, eps, residual=lr)
    y, h = out if residual else (out, None)
    h64, rstd, y64 = _reference(x, r, w, eps)
    _check(y, y64, 48 * E32 * y64.abs(), dt, "y")
    leaves = [lx, lw] + ([lr] if residual else [])
    if residual:
        _check(h, h64, E32 * h64.abs(), dt, "h")
        got = torch.autograd.grad((y, h), leaves, (g.to(device), gh.to(device)))
        assert torch.equal(got[0], got[2])
    else:
        got = torch.autograd.grad(y, leaves, g.to(device))
    g64, u64 = g.double(), g.double() * w.double()
    dot, dot_abs = (u64 * h64).mean(-1, keepdim=True), (u64 * h64).abs().mean(-1, keepdim=True)
    f = rstd ** 2 * dot
    dx = rstd * (u64 - h64 * f) + (gh.double() if residual else 0)
    e = _u(dt) + 48 * E32
    bx = rstd * (8 * E32 * u64.abs() + h64.abs() * (e * f.abs() + rstd ** 2 * dot_abs * e * 2)) \
        + (48 + 8) * E32 * rstd * (u64.abs() + (h64 * f).abs()) + 2 * E32 * dx.abs()
    _check(got[0], dx, bx, dt, "dx")
    terms = g64 * h64 * rstd
    _check(got[1], terms.sum(0), terms.abs().sum(0) * (e + (rows + 8) * E32), dt, "dw")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,n", [(5000, 128), (3001, 40), (1500, 2048), (700, 8192)])
def test_many_rows(rows, n, dt, device):
    """More rows than the backward has workgroups: dw sums over rows of one workgroup and over workgroups."""
    from maloq_amd.norm import rms_norm
    x, r, w, g, gh = _inputs(rows, n, dt, seed=rows)
    lx, lw = (t.to(device).requires_grad_() for t in (x, w))
    y, h = rms_norm(lx, lw, 1e-6, residual=r.to(device))
    gx, gw = torch.autograd.grad((y, h), (lx, lw), (g.to(device), gh.to(device)))
    h64, rstd, y64 = _reference(x, r, w, 1e-6)
    _check(y, y64, 48 * E32 * y64.abs(), dt, "y")
    terms = g.double() * h64 * rstd
    e = _u(dt) + 48 * E32
    _check(gw, terms.sum(0), terms.abs().sum(0) * (e + (rows + 8) * E32), dt, "dw")
    again = torch.autograd.grad(rms_norm(lx, lw, 1e-6, residual=r.to(device)), (lx, lw), (g.to(device), gh.to(device)))
    assert torch.equal(again[0], gx) and torch.equal(again[1], gw)


def test_gradient_against_differences(device):
    """<gradient, d> beside (L(t + e d) - L(t - e d)) / 2 e of L = sum(c y + c' h), in fp32: e = 2^-7
    leaves e^2 / 6 of the third derivative (of size 10 at most here) and 2^-24 of L's terms over e."""
    from maloq_amd.norm import rms_norm
    x, r, w, c, ch = (t.to(device) for t in _inputs(33, 160, torch.float32, seed=4))
    d, dw = torch.randn_like(x), torch.randn_like(w)

    def loss(e):
        y, h = rms_norm(x + e * d, w + e * dw, 1e-6, residual=r)
        return (y.double() * c).sum() + (h.double() * ch).sum()

    lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(rms_norm(lx, lw, 1e-6, residual=r), (lx, lw), (c, ch))
    want = (gx.double() * d).sum() + (gw.double() * dw).sum()
    got = (loss(2.0 ** -7) - loss(-2.0 ** -7)) * 2.0 ** 6
    size = (gx.double() * d).abs().sum() + (gw.double() * dw).abs().sum()
    assert abs(got - want) <= size * 2.0 ** -9


@pytest.mark.parametrize("dt", TYPES)
def test_strides_and_broadcasts(dt, device):
    from maloq_amd.norm import rms_norm
    gen = torch.Generator().manual_seed(1)
    base = torch.randn(9, 5, 72, generator=gen).to(dt).to(device)
    w = torch.ones(64, device=device, dtype=dt) + torch.arange(64, device=device).to(dt) / 64
    views = {"offset columns": base[..., 3:67], "aligned columns": base[..., 8:72], "every other row": base[:, ::2, :64],
             "transposed rows": base[..., :64].transpose(0, 1), "expanded": base[:1, :1, :64].expand(9, 5, 64),
             "across": base.permute(1, 2, 0)[:, :64, :].transpose(1, 2)}
    for name, v in views.items():
        c = v.contiguous()
        assert torch.equal(rms_norm(v, w), rms_norm(c, w)), name
        y, h = rms_norm(c, w, residual=v)
        y2, h2 = rms_norm(c, w, residual=c.clone())
        assert torch.equal(y, y2) and torch.equal(h, h2), name
        lv = v.detach().requires_grad_()
        lr = torch.zeros(64, device=device, dtype=dt, requires_grad=True)  # one row for all: its gradient is the sum
        y, h = rms_norm(lv, w, residual=lr.expand(v.shape))
        gx, gr = torch.autograd.grad((y, h), (lv, lr), (v, v))
        torch.testing.assert_close(gr, gx.reshape(-1, 64).sum(0), rtol=2 ** -7, atol=2 ** -4)
        # gradients that are views: expanded, as of a sum, and across
        ones = torch.ones((), device=device, dtype=dt).expand(v.shape)
        a, = torch.autograd.grad(rms_norm(lv, w), lv, ones)
        b, = torch.autograd.grad(rms_norm(lv, w), lv, ones.contiguous())
        assert torch.equal(a, b), name


@pytest.mark.parametrize("dt", TYPES)
def test_edges(dt, device):
    from maloq_amd.norm import rms_norm, rms_norm_quantized
    w = torch.ones(128, device=device, dtype=dt, requires_grad=True)
    # no rows
    x = torch.zeros(0, 128, device=device, dtype=dt, requires_grad=True)
    y = rms_norm(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == gx.shape == (0, 128) and not gw.any()
    assert rms_norm_quantized(x.detach(), w)[1].shape == (0,)
    # a row of zeros; a row with a NaN; one with an infinity: only their own rows
    x = torch.randn(5, 128, device=device).to(dt)
    x[1] = 0
    x[2, 3] = float("nan")
    x[3, 4] = float("inf")
    clean = torch.randn(5, 128, device=device).to(dt)
    clean[0], clean[4] = x[0], x[4]
    y, yc = rms_norm(x, w), rms_norm(clean, w)
    assert torch.equal(y[0], yc[0]) and torch.equal(y[4], yc[4])
    assert not y[1].any() and y[2].isnan().all() and y[3, 4].isnan() and not y[3, :4].any()
    q, scale = rms_norm_quantized(x, w)
    qc, sc = rms_norm_quantized(clean, w)
    assert torch.equal(q[0].float(), qc[0].float()) and torch.equal(scale[4], sc[4])
    assert scale[2].isnan() and scale[3].isnan() and not q[1].float().any() and scale[1] == 2.0 ** -100 / 448
    # only one of the two outputs is used
    lx, lr = (torch.randn(4, 128, device=device).to(dt).requires_grad_() for _ in range(2))
    y, h = rms_norm(lx, w, residual=lr)
    gh, = torch.autograd.grad(h, lr, torch.ones_like(h), retain_graph=True)
    assert bool((gh == 1).all())
    a = torch.autograd.grad(y, (lx, lr, w), torch.ones_like(y), retain_graph=True)
    b = torch.autograd.grad((y, h), (lx, lr, w), (torch.ones_like(y), torch.zeros_like(h)))
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def _e4m3_bound(y64, scale):
    """Half a step of e4m3 at every value: 2^-4 of it, 2^-10 of the scale at the least."""
    return torch.maximum(y64.abs() * 2.0 ** -4, scale * 2.0 ** -10)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [1, 8, 97, 128, 1000, 4096, 5001, 16384])
def test_eight_bits(n, dt, device):
    from maloq_amd.dense import quantize_rows
    from maloq_amd.norm import rms_norm_quantized
    x, r, w, _, _ = _inputs(7, n, dt, seed=n)
    q, scale, h = rms_norm_quantized(x.to(device), w.to(device), 1e-6, residual=r.to(device))
    h64, _, y64 = _reference(x, r, w, 1e-6)
    _check(h, h64, E32 * h64.abs(), dt, "h")
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (7,)
    s = scale.double().cpu()[:, None]
    assert bool(((s * 448 - y64.abs().amax(-1, keepdim=True)).abs() <= 50 * E32 * s * 448).all())
    err = (q.double().cpu() * s - y64).abs()
    assert bool((err <= _e4m3_bound(y64, s) * (1 + 2.0 ** -10) + 50 * E32 * y64.abs()).all())
    # whole numbers up to 7 (448 = 7 x 64: a scale of a power of two) come back as they are
    k = torch.randint(-7, 8, (7, n)).to(dt)
    k[:, 0] = 7
    q, scale = quantize_rows((k * 0.25).to(device))
    assert torch.equal(q.float().cpu() * scale.cpu()[:, None], k.float() * 0.25)


def test_refusals(device):
    from maloq_amd.dense import quantize_rows
    from maloq_amd.norm import rms_norm, rms_norm_quantized
    x, w = torch.zeros(3, 64, device=device), torch.ones(64, device=device)
    for bad in (lambda: rms_norm(x, w[:32]), lambda: rms_norm(x, w.half()), lambda: rms_norm(x.double(), w.double()),
                lambda: rms_norm(x, w, residual=x[:2]), lambda: rms_norm(x, w, residual=x.bfloat16()),
                lambda: rms_norm(x, w.cpu()), lambda: rms_norm(x.cpu(), w.cpu()), lambda: rms_norm(x[:, :0], w[:0]),
                lambda: rms_norm(torch.zeros(1, 16385, device=device), torch.ones(16385, device=device)),
                lambda: rms_norm_quantized(x.int(), w), lambda: quantize_rows(x.cpu()),
                lambda: quantize_rows(torch.zeros(1, 16385, device=device))):
        with pytest.raises(ValueError):
            bad()
    lx = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(rms_norm(lx, w), lx, torch.ones_like(x), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(rms_norm(lx, w), lx, torch.ones(2, 3, 64, device=device), is_grads_batched=True)
