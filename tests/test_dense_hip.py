"""Linear layers with their epilogue (maloq_amd.dense) against 64 bits, training and in 8 bits.

Bounds, each value for itself: an fp32 sum of k products is off by at most (k + 8) 2^-24 of the sum
of their magnitudes; an activation adds 2^-20 (1 + |z|) of the result (a hardware exponential and
reciprocal, 16-bit results) and passes on its argument's error times at most 1.13; the result is
rounded once (u = eps / 2 of the value).  Gradients: the stored argument is off by u, which the
slope takes times at most 0.8; the slope's product with the gradient is rounded once more before
the products.  fp32 products are six of split floats: 2-norms, as for the framework's others.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALVES = [torch.bfloat16, torch.float16]
E32 = 2.0 ** -24
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
# rows, inner, outer: single values, single rows, edges of vectors, tiles of 128 and 256, the
# contraction's steps of 32 and 64 and its parts
SIZES = [(1, 1, 1), (1, 8, 8), (1, 300, 1), (2, 7, 9), (3, 64, 40), (16, 32, 256), (17, 70, 90), (33, 4096, 64),
         (100, 33, 8), (128, 128, 128), (129, 130, 131), (255, 96, 257), (300, 1000, 129), (31, 2056, 520)]
LARGE = [(4100, 72, 3588), (3900, 40, 4001)]
ACTS = ["none", "relu", "silu", "gelu"]


def _u(dt):
    return torch.finfo(dt).eps / 2


def _inputs(m, k, n, dt, seed=0):
    gen = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=gen).to(dt)
    return make(m, k), (make(n, k).float() / math.sqrt(k)).to(dt), make(n), make(m, n), make(m, n)


def _act(z, act):
    return {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu,
            "gelu": torch.nn.functional.gelu}[act](z)


def _slope(z, act):
    z = z.clone().requires_grad_()
    return torch.autograd.grad(_act(z, act).sum(), z)[0] if act != "none" else torch.ones_like(z)


def _check(got, ref, bound, what):
    dt = got.dtype
    err = (got.double() - ref).abs()
    lim = bound + _u(dt) * ref.abs() + TINY[dt]
    assert bool((err <= lim * (1 + 1e-6)).all()), (what, (err / lim.clamp_min(1e-300)).max().item())


def _forward_bound(a, w, z, y, k):
    return 1.13 * (k + 8) * E32 * (a.abs() @ w.abs().T) + 2.0 ** -20 * (1 + z.abs()) * y.abs() + 2 * E32 * y.abs()


def _run(m, k, n, dt, act, bias, residual, device, seed=0):
    from maloq_amd.dense import linear_act
    x, w, b, r, g = (t.to(device) for t in _inputs(m, k, n, dt, seed))
    b, r = b if bias else None, r if residual else None
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    args = [next(it) if t is not None else None for t in (x, w, b, r)]
    y = linear_act(args[0], args[1], args[2], act=act, residual=args[3])
    grads = iter(torch.autograd.grad(y, leaves, g))
    gx, gw, gb, gr = (next(grads) if t is not None else None for t in (x, w, b, r))
    with torch.no_grad():
        assert torch.equal(linear_act(x, w, b, act=act, residual=r), y)
    d = [t.double() if t is not None else None for t in (x, w, b, r, g)]
    z = d[0] @ d[1].T + (d[2] if bias else 0)
    y64 = _act(z, act) + (d[3] if residual else 0)
    return (y, gx, gw, gb, gr), d, z, y64


@pytest.mark.parametrize("dt", HALVES)
@pytest.mark.parametrize("m,k,n,act", [(*s, a) for s in SIZES for a in ACTS] + [(*s, a) for s in LARGE for a in ("none", "gelu")])
def test_sixteen_bits(m, k, n, act, dt, device):
    bias, residual = (m + n) % 3 > 0, (k + n) % 2 > 0
    (y, gx, gw, gb, gr), (x, w, b, r, g), z, y64 = _run(m, k, n, dt, act, bias, residual, device, seed=m + n)
    pre = y64 - (r if residual else 0)
    bz = (k + 8) * E32 * (x.abs() @ w.abs().T + (b.abs() if bias else 0))
    _check(y, y64, 1.13 * bz + 2.0 ** -20 * (1 + z.abs()) * pre.abs() + 2 * E32 * y64.abs(), "y")
    dz = g * _slope(z, act)
    ez = 0.8 * g.abs() * (_u(dt) * z.abs() + bz + TINY[dt]) + 2.0 ** -20 * (1 + z.abs()) * g.abs() if act != "none" else 0 * g
    if act == "relu":  # a slope of 0 or 1, but where the argument's sign is within its error
        ez = g.abs() * (z.abs() <= bz + TINY[dt])
    er = ez + (_u(dt) * dz.abs() + TINY[dt] if act != "none" else 0)
    _check(gx, dz @ w, er @ w.abs() + (n + 8) * E32 * (dz.abs() @ w.abs()), "dx")
    _check(gw, dz.T @ x, er.T @ x.abs() + (m + 8) * E32 * (dz.abs().T @ x.abs()), "dw")
    if bias:
        _check(gb, dz.sum(0), ez.sum(0) + (m + 8) * E32 * dz.abs().sum(0), "db")
    if residual:
        assert torch.equal(gr.double(), g)


def _tol(n):
    """2-norm of n products of split floats (the framework's other fp32 products)."""
    return 4 * (2.0 ** -23 + math.sqrt(3 * n / 8) * 2.0 ** -25)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,k,n", SIZES + LARGE[:1])
def test_fp32(m, k, n, act, device):
    bias, residual = (m + n) % 3 > 0, (k + n) % 2 > 0
    (y, gx, gw, gb, gr), (x, w, b, r, g), z, y64 = _run(m, k, n, torch.float32, act, bias, residual, device, seed=m + n)
    # the norms that a product's error goes by: of the magnitudes' product
    size = lambda p, q: (p.square() @ q.square()).sum().sqrt()
    off = lambda a, t: (a.double() - t).norm()
    ez = _tol(k) * size(x, w.T) + 8 * E32 * z.norm()
    assert off(y, y64) <= 1.13 * ez + 8 * E32 * ((1 + z.abs()) * y64).norm() + 2 * E32 * y64.norm()
    dz = g * _slope(z, act)
    gmax = g.abs().max()
    ed = gmax * (0.8 * ez + E32 * z.norm()) + 16 * E32 * ((1 + z.abs()) * g).norm() if act != "none" else 0
    if act == "relu":
        near = z.abs() <= 16 * (k + 8) * E32 * (x.abs() @ w.abs().T + 1)
        ed = (g * near).norm()
    op = lambda t: torch.linalg.matrix_norm(t, 2)
    assert off(gx, dz @ w) <= _tol(n) * size(dz, w) + ed * op(w) + 1e-300
    assert off(gw, dz.T @ x) <= _tol(m) * size(dz.T, x) + ed * op(x) + 1e-300
    if bias:
        assert off(gb, dz.sum(0)) <= (m + 8) * E32 * dz.abs().sum(0).norm() + ed * math.sqrt(m)
    if residual:
        assert torch.equal(gr.double(), g)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k,n", SIZES + LARGE)
def test_eight_bits(m, k, n, out, device):
    """The product of the e4m3 numbers as they are (their rounding is the quantiser's).  The matrix unit
    aligns the 64 products of an instruction to the largest: 2^-11 of that one is left out at most."""
    from maloq_amd.dense import linear_quantized, quantize_rows
    act = ACTS[(m + n) % 4]
    x, w, b, r, _ = (t.to(device) for t in _inputs(m, k, n, torch.float32, seed=k))
    b, r = b.to(out), r.to(out)
    (q, s), (p, t) = quantize_rows(x), quantize_rows(w)
    y = linear_quantized(q, s, p, t, b, act=act, residual=r, dtype=out)
    a64, w64 = q.double() * s.double()[:, None], p.double() * t.double()[:, None]
    z = a64 @ w64.T + b.double()
    pre = _act(z, act)
    unit = 2.0 ** -11 * ((k + 63) // 64) * a64.abs().amax(1)[:, None] * w64.abs().amax(1)
    bz = unit + (k + 8) * E32 * (a64.abs() @ w64.abs().T) + 2 * E32 * b.double().abs()
    _check(y, pre + r.double(), 1.13 * bz + 2.0 ** -20 * (1 + z.abs()) * pre.abs() + 2 * E32 * (pre.abs() + r.double().abs()), "y")


@pytest.mark.parametrize("m,k,n", SIZES + LARGE)
def test_eight_bits_exactly(m, k, n, device):
    """Numbers of 1/8 to 15/8 in steps of 1/8, scales that are powers of two: every sum is exact."""
    from maloq_amd.dense import linear_quantized
    gen = torch.Generator().manual_seed(m + k)
    q, p = ((torch.randint(-15, 16, s, generator=gen) / 8).to(torch.float8_e4m3fn).to(device) for s in ((m, k), (n, k)))
    s, t = (torch.exp2(torch.randint(-3, 4, (c,), generator=gen).float()).to(device) for c in (m, n))
    b, r = ((torch.randint(-64, 65, c, generator=gen) / 8).to(device) for c in ((n,), (m, n)))
    y = linear_quantized(q, s, p, t, b, act="relu", residual=r, dtype=torch.float32)
    assert torch.equal(y.double(), torch.relu((q.double() @ p.double().T) * s.double()[:, None] * t.double() + b.double()) + r.double())


@pytest.mark.parametrize("dt", HALVES + [torch.float32])
@pytest.mark.parametrize("act", ["silu", "gelu", "none"])
def test_gradient_against_differences(dt, act, device):
    """<gradient, d> beside (L(t + e d) - L(t - e d)) / 2 e.  L in fp32 (the operator's own fp32 form on
    the same values): e = 2^-6 leaves e^2 / 6 of the third derivative; 16-bit gradients are off by 3 u."""
    from maloq_amd.dense import linear_act
    x, w, b, r, c = (t.to(device) for t in _inputs(40, 56, 72, dt, seed=9))
    dirs = [torch.randn_like(t.float()) for t in (x, w, b)]

    def loss(e):
        a = [t.float() + e * d for t, d in zip((x, w, b), dirs)]
        return (linear_act(*a, act=act).double() * c.double()).sum()

    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(linear_act(*leaves, act=act), leaves, c)
    terms = [(g.double() * d.double()) for g, d in zip(got, dirs)]
    want, size = sum(t.sum() for t in terms), sum(t.abs().sum() for t in terms)
    e = 2.0 ** -6
    assert abs((loss(e) - loss(-e)) / (2 * e) - want) <= size * (2.0 ** -9 + 3 * _u(dt))


@pytest.mark.parametrize("dt", HALVES + [torch.float32])
def test_strides_and_broadcasts(dt, device):
    from maloq_amd.dense import linear_act
    gen = torch.Generator().manual_seed(2)
    base = torch.randn(6, 10, 80, generator=gen).to(dt).to(device)
    wide = (torch.randn(48, 80, generator=gen) / 8).to(dt).to(device)
    views = {"offset columns": (base[..., 3:67], wide[:, 5:69]), "aligned columns": (base[..., 8:72], wide[:, 16:80]),
             "every other row": (base[:, ::2, :64], wide[::2, :64]),
             "transposed rows": (base[..., :64].transpose(0, 1), wide[:, :64]),
             "across": (base.permute(1, 2, 0).transpose(1, 2)[..., :64], wide[:, :64].t().contiguous().t()),
             "expanded": (base[:1, :1, :64].expand(6, 10, 64), wide[:1, :64].expand(48, 64)),
             "one row": (base[0, 0, :64], wide[:, :64])}
    for name, (x, w) in views.items():
        lx, lw = x.detach().requires_grad_(), w.detach().requires_grad_()
        cx, cw = x.contiguous().requires_grad_(), w.contiguous().requires_grad_()
        n = w.shape[0]
        lr = torch.randn(n, generator=gen).to(dt).to(device).requires_grad_()  # a residual of one row for all
        y, yc = linear_act(lx, lw, act="silu", residual=lr.expand(*x.shape[:-1], n)), linear_act(cx, cw, act="silu")
        assert y.shape == (*x.shape[:-1], n), name
        torch.testing.assert_close(y.float(), (yc.float() + lr.float()), rtol=2 * torch.finfo(dt).eps, atol=4 * torch.finfo(dt).eps)
        g = torch.randn(n, *x.shape[:-1], generator=gen).to(dt).to(device).movedim(0, -1)  # across
        got = torch.autograd.grad(y, (lx, lw, lr), g)
        want = torch.autograd.grad(yc, (cx, cw), g.contiguous())
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), name
        torch.testing.assert_close(got[2], g.reshape(-1, n).sum(0) if x.dim() > 1 else g, rtol=2 ** -6, atol=2 ** -5)
        ones = torch.ones((), device=device, dtype=dt).expand(yc.shape)  # the gradient of a sum
        a = torch.autograd.grad(linear_act(cx, cw, act="gelu"), (cx, cw), ones)
        b = torch.autograd.grad(linear_act(cx, cw, act="gelu"), (cx, cw), ones.contiguous())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), name


@pytest.mark.parametrize("dt", HALVES + [torch.float32])
def test_needs(dt, device):
    """Each set of wanted gradients gives what all of them together give."""
    from maloq_amd.dense import linear_act
    x, w, b, r, g = (t.to(device) for t in _inputs(50, 36, 44, dt, seed=3))

    def grads(needs):
        leaves = [t.clone().requires_grad_(n) for t, n in zip((x, w, b, r), needs)]
        y = linear_act(*leaves[:3], act="silu", residual=leaves[3])
        return torch.autograd.grad(y, [t for t in leaves if t.requires_grad], g)

    full = grads((True,) * 4)
    for bits in range(1, 15):
        needs = [bool(bits >> i & 1) for i in range(4)]
        assert all(torch.equal(a, f) for a, f in zip(grads(needs), [f for f, n in zip(full, needs) if n])), needs


@pytest.mark.parametrize("dt", HALVES + [torch.float32])
def test_not_finite(dt, device):
    """NaN and infinities stay in the rows and columns that they belong to; relu keeps NaN."""
    from maloq_amd.dense import linear_act
    x, w, b, r, _ = (t.to(device) for t in _inputs(140, 96, 150, dt, seed=5))
    clean = linear_act(x, w, b, act="relu")
    y = x.clone()
    y[7, 5], y[139, 95] = float("nan"), float("inf")
    v = w.clone()
    v[149, 0] = -float("inf")
    got = linear_act(y, v, b, act="none")
    ref = torch.nn.functional.linear(y.cpu().double(), v.cpu().double(), b.cpu().double())
    assert torch.equal(got.isnan().cpu(), ref.isnan()) and torch.equal(got.isposinf().cpu(), ref.isposinf())
    assert torch.equal(got.isneginf().cpu(), ref.isneginf())
    keep = [i for i in range(140) if i not in (7, 139)]
    assert torch.equal(linear_act(y, w, b, act="relu")[keep], clean[keep])
    assert linear_act(y, w, b, act="relu")[7].isnan().all()


def test_no_rows_no_inner_no_outer(device):
    from maloq_amd.dense import linear_act, linear_quantized, quantize_rows
    for dt in HALVES + [torch.float32]:
        b = torch.randn(24, device=device).to(dt).requires_grad_()
        for m, k, n in ((0, 16, 24), (5, 0, 24), (5, 16, 0)):
            x, w = (torch.randn(*s, device=device).to(dt).requires_grad_() for s in ((m, k), (n, k)))
            y = linear_act(x, w, b[:n], act="silu")
            assert torch.equal(y, torch.nn.functional.silu(torch.nn.functional.linear(x.float(), w.float(), b[:n].float())).to(dt)) \
                or y.numel() and k == 0
            gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
            assert gx.shape == x.shape and gw.shape == w.shape
            assert not gx.any() and not gw.any()
            if m == 0:
                assert not gb.any()
    q, s = quantize_rows(torch.randn(0, 32, device=device))
    p, t = quantize_rows(torch.randn(8, 32, device=device))
    assert linear_quantized(q, s, p, t).shape == (0, 8)


def test_refusals(device):
    from maloq_amd.dense import linear_act, linear_quantized, quantize_rows
    x, w, b = torch.zeros(3, 64, device=device), torch.zeros(40, 64, device=device), torch.zeros(40, device=device)
    r = torch.zeros(3, 40, device=device)
    for bad in (lambda: linear_act(x, w, act="tanh"), lambda: linear_act(x, w[:, :32]), lambda: linear_act(x, w.half()),
                lambda: linear_act(x, w, b[:39]), lambda: linear_act(x, w, b.bfloat16()), lambda: linear_act(x, w, residual=r[:2]),
                lambda: linear_act(x, w, residual=r.half()), lambda: linear_act(x.double(), w.double()),
                lambda: linear_act(x, w.cpu()), lambda: linear_act(x.cpu(), w.cpu()), lambda: linear_act(x, w[0])):
        with pytest.raises(ValueError):
            bad()
    (q, s), (p, t) = quantize_rows(x), quantize_rows(w)
    for bad in (lambda: linear_quantized(x, s, p, t), lambda: linear_quantized(q, s, w, t), lambda: linear_quantized(q, s[:2], p, t),
                lambda: linear_quantized(q, s, p, t.half()), lambda: linear_quantized(q, s, p, t, b),
                lambda: linear_quantized(q, s, p, t, dtype=torch.float64), lambda: linear_quantized(q, s, p[:, :32], t)):
        with pytest.raises(ValueError):
            bad()
    lx = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(linear_act(lx, w), lx, torch.ones_like(r), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(linear_act(lx, w), lx, torch.ones(2, 3, 40, device=device), is_grads_batched=True)
