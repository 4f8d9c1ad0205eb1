"""Group norm with an activation, channels last (maloq_amd.norm.group_norm), against 64 bits.

Bounds, each value for itself.  A sum is a chain of at most L fp32 additions: 64 where a workgroup holds a group's values (eight
places, eight channels, six shuffles, 16 rows and 16 columns in LDS), and of several launches three operations more for each batch
of eight places of a thread.  With A the mean magnitude of a group's values, its mean is off by L 2^-24 A and its deviation by
(L + 4) 2^-24 of itself; the normed value, the activation's argument and the gradients pass these on as their formulas say; the
slope of an activation takes its argument's error times 0.8, its value times 1.13; results are rounded once.
"""
import ctypes
import math

import pytest
import torch

from test_dense_hip import ACTS, E32, TINY, _act, _slope, _u

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# samples, places, channels, groups: single values, groups of any size, many samples of few values, registers of one wave to
# sixteen, parts of a group's places, groups wider than a tile
SIZES = [(1, 1, 1, 1), (1, 1, 8, 1), (2, 3, 6, 2), (3, 16, 64, 8), (5, 777, 330, 11), (1, 1, 8192, 1), (3, 2, 5000, 1), (300, 1, 512, 16),
         (2000, 2, 40, 5), (2, 100, 1000, 1), (1, 5000, 24, 24), (2, 9000, 33, 3), (64, 50, 256, 256), (4, 300, 4096, 1), (7, 5, 9000, 2),
         (2, 1000, 128, 8), (1, 40000, 8, 2), (1, 4096, 512, 32), (2, 600, 1030, 2), (1, 1, 20000, 1), (3, 8, 512, 1), (1, 30000, 2, 1), (70, 1, 4096, 1), (9, 256, 256, 8),
         (5000, 1, 128, 8), (333, 3, 30, 5), (1001, 4, 8, 1), (2, 4, 8192, 8192), (3, 1, 9000, 9000), (257, 2, 12, 12), (4099, 1, 7, 7)]


def _inputs(n, p, c, dt, seed=0, mean=1.0):
    gen = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=gen)
    x = make(n, p, c) * (1 + 0.3 * make(c)) + mean * make(c)
    return [t.to(dt) for t in (x, 1 + 0.2 * make(c), 0.2 * make(c), make(n, p, c))]


def _plan(dt, n, p, c, groups, backward):
    from maloq_amd import _lib
    plan = (ctypes.c_int64 * 8)()
    code = TYPES.index(dt)
    _lib.call("maloq_group_norm_plan", code, n, p, c, groups, int(backward), ctypes.cast(plan, ctypes.c_void_p).value)
    return list(plan)


def _steps(dt, n, p, c, groups):
    """L"""
    held = all(_plan(dt, n, p, c, groups, b)[0] for b in (0, 1))
    return 64 if held else 96 + 3 * math.ceil(p / 8)


def _check(got, ref, bound, what):
    dt = got.dtype
    err = (got.double() - ref).abs()
    lim = bound + _u(dt) * ref.abs() + TINY[dt]
    assert bool((err <= lim * (1 + 1e-6)).all()), (what, (err / lim.clamp_min(1e-300)).max().item())


def _reference(x, w, b, g, groups, act, dt, steps, eps=1e-5):
    """{name: (value, bound without the last rounding)} in 64 bits."""
    n, p, c = x.shape
    x, g = (t.double().view(n, p, groups, -1) for t in (x, g))
    w, b = (t.double().view(groups, -1) for t in (w, b))
    over = lambda t: t.mean((1, 3), keepdim=True)
    L = steps * E32
    mean = over(x)
    rstd = (over((x - mean).square()) + eps).rsqrt()
    nx = (x - mean) * rstd
    en = rstd * L * over(x.abs()) + nx.abs() * (L + 4 * E32)
    z = nx * w + b
    ez = w.abs() * en + 2 * E32 * (z.abs() + b.abs())
    y = _act(z, act)
    out = {"y": (y, 1.13 * ez + 2.0 ** -20 * (1 + z.abs()) * y.abs())}
    u = g * _slope(z, act)
    eu = 0 * g if act == "none" else g.abs() * (z.abs() <= ez) if act == "relu" else g.abs() * (0.8 * ez + 2.0 ** -20 * (1 + z.abs()))
    uw, euw = u * w, (eu + E32 * u.abs()) * w.abs()
    m0, m1 = over(uw), over(uw * nx)
    e0 = over(euw) + L * over(uw.abs())
    e1 = over(euw * nx.abs() + uw.abs() * en) + L * over((uw * nx).abs())
    dx = rstd * (uw - m0 - nx * m1)
    out["dx"] = (dx, rstd * (euw + e0 + en * m1.abs() + nx.abs() * e1 + 4 * E32 * (uw.abs() + m0.abs() + (nx * m1).abs())) + dx.abs() * (L + 4 * E32))
    every = (steps + n) * E32
    out["dw"] = ((u * nx).sum((0, 1)), (eu * nx.abs() + u.abs() * en).sum((0, 1)) + every * (u * nx).abs().sum((0, 1)))
    out["db"] = (u.sum((0, 1)), eu.sum((0, 1)) + every * u.abs().sum((0, 1)))
    return {k: tuple(t.reshape(n, p, c) if k in ("y", "dx") else t.reshape(c) for t in v) for k, v in out.items()}


def _run(x, w, b, g, groups, act, eps=1e-5):
    from maloq_amd.norm import group_norm
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
    y = group_norm(leaves[0], groups, leaves[1], leaves[2], eps, act=act)
    return (y, *torch.autograd.grad(y, leaves, g))


@gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,p,c,groups", SIZES)
def test_against_64_bits(n, p, c, groups, dt, device):
    from maloq_amd.norm import group_norm
    for act in ACTS if n * p * c < 200000 else [ACTS[(n + p + c) % 4], "silu"]:
        x, w, b, g = (t.to(device) for t in _inputs(n, p, c, dt, seed=n + c))
        got = _run(x, w, b, g, groups, act)
        ref = _reference(x, w, b, g, groups, act, dt, _steps(dt, n, p, c, groups))
        for t, (name, (value, bound)) in zip(got, ref.items()):
            assert t.dtype == dt
            _check(t, value, bound, (name, act))
        assert torch.equal(group_norm(x, groups, w, b, act=act), got[0])
        assert all(torch.equal(a, e) for a, e in zip(_run(x, w, b, g, groups, act), got))


@gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,p,c,groups", [(2, 64, 48, 3), (1, 5000, 24, 2)])
def test_far_from_zero(n, p, c, groups, dt, device):
    """Means that are many deviations: squares' sums would lose the variance."""
    x, w, b, g = (t.to(device) for t in _inputs(n, p, c, torch.float32, seed=2))
    x = (x * 0.25 + (1000 if dt == torch.float32 else 16)).to(dt)
    w, b, g = w.to(dt), b.to(dt), g.to(dt)
    got = _run(x, w, b, g, groups, "silu")
    for t, (name, (value, bound)) in zip(got, _reference(x, w, b, g, groups, "silu", dt, _steps(dt, n, p, c, groups)).items()):
        _check(t, value, bound, name)


@gpu
@pytest.mark.parametrize("n,p,c,groups", [(2, 64, 48, 3), (1, 9000, 24, 2), (3, 1, 16, 2), (2, 50, 30, 2), (1, 7777, 21, 3), (700, 3, 11, 1)])
def test_constant_groups(n, p, c, groups, device):
    """No deviation: b's activation, and no gradient of x beside rstd = eps^-1/2."""
    for dt in TYPES:
        x = torch.full((n, p, c), 3.0, device=device, dtype=dt)
        _, w, b, g = (t.to(device) for t in _inputs(n, p, c, dt, seed=1))
        y, gx, gw, gb = _run(x, w, b, g, groups, "relu")
        assert torch.equal(y, torch.relu(b).expand(n, p, c)) and bool(gx.isfinite().all()) and not gw.any()


@gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("p,c,groups", [(40, 96, 4), (9000, 40, 2)])
def test_strides(p, c, groups, dt, device):
    gen = torch.Generator().manual_seed(7)
    base = torch.randn(4, p, c + 40, generator=gen).to(dt).to(device)
    w, b = (torch.randn(c + 3, generator=gen).to(dt).to(device) for _ in range(2))
    from maloq_amd.norm import group_norm
    views = {"columns": base[..., 3:3 + c], "every other sample": base[::2, :, :c], "every other place": base[:, ::2, 8:8 + c],
             "one sample": base[1:2, :, :c], "expanded": base[:1, :1, :c].expand(3, 5, c), "no places": base[:, 0, 5:5 + c],
             "across": base[..., :c].permute(0, 2, 1).contiguous().permute(0, 2, 1), "four": base[..., :c].unflatten(1, (-1, 4))}
    for name, x in views.items():
        g = torch.randn(*x.shape[1:], x.shape[0], generator=gen).to(dt).to(device).movedim(-1, 0)  # across
        leaves, plain = [x.detach().requires_grad_(), w[3:].detach().requires_grad_(), b[1:c + 1].detach().requires_grad_()], None
        y = group_norm(leaves[0], groups, leaves[1], leaves[2], act="gelu")
        got = torch.autograd.grad(y, leaves, g)
        flat = x.contiguous().view(x.shape[0], -1, c)
        plain = _run(flat, w[3:].contiguous(), b[1:c + 1].contiguous(), g.contiguous().view_as(flat), groups, "gelu")
        assert y.shape == x.shape and torch.equal(y.reshape(flat.shape), plain[0]), name
        assert torch.equal(got[0].reshape(flat.shape), plain[1]) and torch.equal(got[1], plain[2]) and torch.equal(got[2], plain[3]), name
        ones = torch.ones((), device=device, dtype=dt).expand(y.shape)
        y = group_norm(leaves[0], groups, leaves[1], leaves[2], act="silu")
        assert torch.equal(torch.autograd.grad(y, leaves[0], ones, retain_graph=True)[0], torch.autograd.grad(y, leaves[0], ones.contiguous())[0]), name


@gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,p,c,groups", [(6, 20, 48, 3), (2, 6000, 40, 2)])
def test_needs_and_defaults(n, p, c, groups, dt, device):
    from maloq_amd.norm import group_norm
    x, w, b, g = (t.to(device) for t in _inputs(n, p, c, dt, seed=3))

    def grads(needs, use=(True, True)):
        leaves = [t.clone().requires_grad_(k) for t, k in zip((x, w, b), needs)]
        y = group_norm(leaves[0], groups, leaves[1] if use[0] else None, leaves[2] if use[1] else None, act="silu")
        wanted = [t for t, k, given in zip(leaves, needs, (True, *use)) if k and given]
        return y, torch.autograd.grad(y, wanted, g)

    y, full = grads((True,) * 3)
    for bits in range(1, 7):
        needs = [bool(bits >> i & 1) for i in range(3)]
        assert all(torch.equal(a, f) for a, f in zip(grads(needs)[1], [f for f, k in zip(full, needs) if k])), needs
    w.fill_(1)
    ones = grads((True,) * 3)
    assert all(torch.equal(a, e) for a, e in zip(grads((True, False, True), (False, True))[1], (ones[1][0], ones[1][2])))
    b.fill_(0)
    ones = grads((True,) * 3)
    assert torch.equal(grads((True, True, False), (True, False))[1][1], ones[1][1])
    bare = grads((True, False, False), (False, False))
    assert torch.equal(bare[0], ones[0]) and torch.equal(bare[1][0], ones[1][0])


@gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("p", [50, 9000])
def test_not_finite(dt, p, device):
    """NaN and infinities stay in their sample's group."""
    x, w, b, g = (t.to(device) for t in _inputs(3, p, 48, dt, seed=5))
    clean = _run(x, w, b, g, 3, "silu")
    bad = x.clone()
    bad[0, 7, 3], bad[2, p - 1, 47] = math.nan, math.inf
    got = _run(bad, w, b, g, 3, "silu")
    hit = torch.zeros(3, p, 48, dtype=torch.bool, device=device)
    hit[0, :, :16] = hit[2, :, 32:] = True
    for a, e in zip(got[:2], clean[:2]):
        assert bool(a[hit].isnan().all()) and torch.equal(a[~hit], e[~hit])
    for a, e in zip(got[2:], clean[2:]):
        assert bool(a[:16].isnan().all()) and bool(a[32:].isnan().all()) and torch.equal(a[16:32], e[16:32])


@gpu
@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_gradient_against_differences(act, device):
    """<gradient, d> beside (L(t + e d) - L(t - e d)) / 2 e in fp32: e = 2^-7 leaves e^2 / 6 of the third derivative along
    directions of unit size beside deviations of about one: 2^-9 of the terms' magnitudes covers it and the sums' rounding."""
    from maloq_amd.norm import group_norm
    x, w, b, c = (t.to(device) for t in _inputs(3, 30, 24, torch.float32, seed=9))
    dirs = [torch.randn_like(t) for t in (x, w, b)]
    got = _run(x, w, b, c, 4, act)[1:]

    def loss(e):
        return (group_norm(*(x + e * dirs[0], 4, w + e * dirs[1], b + e * dirs[2]), act=act).double() * c.double()).sum()

    terms = [g.double() * d.double() for g, d in zip(got, dirs)]
    want, size = sum(t.sum() for t in terms), sum(t.abs().sum() for t in terms)
    e = 2.0 ** -7
    assert abs((loss(e) - loss(-e)) / (2 * e) - want) <= size * 2.0 ** -9


@gpu
def test_empty(device):
    from maloq_amd.norm import group_norm
    for dt in TYPES:
        for sizes in ((0, 5, 16), (3, 0, 16), (0, 16), (2, 4, 0, 16)):
            x, w, b = (torch.zeros(*s, device=device, dtype=dt).requires_grad_() for s in (sizes, (16,), (16,)))
            y = group_norm(x, 4, w, b, act="silu")
            gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
            assert y.shape == sizes and gx.shape == sizes and not gw.any() and not gb.any()


@gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,p,c,groups", [(1, 16, 64, 8), (3, 500, 96, 4), (2, 9000, 64, 2)])
def test_captured_and_on_another_stream(n, p, c, groups, dt, device):
    from maloq_amd.norm import group_norm
    x, w, b, g = (t.to(device) for t in _inputs(n, p, c, dt, seed=1))
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def work():
        y = group_norm(x, groups, w, b, act="gelu")
        return (y.detach(), *torch.autograd.grad(y, leaves, g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, e) for a, e in zip(first, work()))
    del first
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in (2, 3, 4):
        with torch.no_grad():
            for t, f in zip((x, w, b, g), _inputs(n, p, c, dt, seed=seed)):
                t.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        assert all(torch.equal(a, e) for a, e in zip(kept, work())), seed


@gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,p,c,groups", [(3, 20, 45, 5), (2, 6000, 40, 2)])
def test_hooks_and_transforms(n, p, c, groups, dt, device):
    from torch.utils.checkpoint import checkpoint
    from maloq_amd.norm import group_norm
    x, w, b, g = (t.to(device) for t in _inputs(n, p, c, dt, seed=4))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    f = lambda: group_norm(x, groups, w, b, act="silu")
    want = torch.autograd.grad(f(), leaves, g)
    for unpack in (lambda t: t.clone(), lambda t: torch.stack([t, t], -1)[..., 0], lambda t: t.movedim(0, -1).contiguous().movedim(-1, 0)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = f()
        assert all(torch.equal(a, e) for a, e in zip(torch.autograd.grad(y, leaves, g), want))
    y = checkpoint(f, use_reentrant=False)
    assert all(torch.equal(a, e) for a, e in zip(torch.autograd.grad(y, leaves, g), want))
    y = torch.compile(lambda *t: group_norm(t[0], groups, t[1], t[2], act="silu"), backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(y, f()) and all(torch.equal(a, e) for a, e in zip(torch.autograd.grad(y, leaves, g), want))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(f(), x, g, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(f(), x, torch.stack([g, g]), is_grads_batched=True)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: group_norm(t, groups))(torch.stack([x.detach()] * 2))


@gpu
def test_opcheck(device):
    from maloq_amd import ops
    for dt in (torch.float16, torch.float32):
        x, w, b, g = (t.to(device) for t in _inputs(3, 20, 24, dt, seed=2))
        stats = ops.group_norm_fwd(x, 4, w, b, 1e-5, 2)[1]
        for op, args in ((ops.group_norm_fwd, (x, 4, w, b, 1e-5, 2)), (ops.group_norm_fwd, (x, 1, None, None, 1e-5, 0)),
                         (ops.group_norm_bwd, (g, x, w, b, stats, 4, 2, True, True)), (ops.group_norm_bwd, (g, x, None, b, stats, 4, 2, False, True)),
                         (ops.group_norm_bwd, (g, x, w, None, stats, 4, 2, True, False))):
            torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


@gpu
def test_refusals(device):
    from maloq_amd import ops
    from maloq_amd.norm import group_norm
    x, w = torch.zeros(3, 5, 24, device=device), torch.zeros(24, device=device)
    stats = torch.zeros(3, 4, 2, device=device)
    for bad in (lambda: group_norm(x, 5, w, w), lambda: group_norm(x, 0, w, w), lambda: group_norm(x, 4, w[:23], w), lambda: group_norm(x, 4, w, w.half()),
                lambda: group_norm(x, 4, w, w, act="tanh"), lambda: group_norm(w, 4), lambda: group_norm(x.double(), 4), lambda: group_norm(x.cpu(), 4),
                lambda: group_norm(x, 4, w.cpu()), lambda: group_norm(x[..., :0], 4), lambda: group_norm(x, 4, x),
                lambda: ops.group_norm_bwd(x[:2], x, w, w, stats, 4, 0, True, True), lambda: ops.group_norm_bwd(x.half(), x, w, w, stats, 4, 0, True, True),
                lambda: ops.group_norm_bwd(x, x, w, w, stats, 8, 0, True, True), lambda: ops.group_norm_bwd(x, x, w, w, stats.half(), 4, 0, True, True)):
        with pytest.raises(ValueError):
            bad()


def test_plans():
    """Every listed size has a plan, and the sizes between them take every way there is."""
    ways, sides = set(), set()
    for dt in TYPES:
        for n, p, c, groups in SIZES:
            for back in (0, 1):
                threads, places, gpt, tiles, parts, sub, slots, span = _plan(dt, n, p, c, groups, back)
                each = c // groups
                if threads:
                    wide = 1
                    while wide * 8 < gpt * each:
                        wide *= 2
                    assert span // wide * places >= p and wide <= span and threads % span == 0 and (span == threads or span <= 64)
                    assert gpt * tiles >= groups and 1 <= slots <= n
                    sides.add((back, span < threads))
                    ways.add((back, threads))
                else:
                    assert parts >= 1 and (sub > 1) == (each > 512) and tiles == (groups * sub if sub > 1 else -(-groups // gpt))
                    ways.add((back, "parts", sub > 1))
    assert ways == {(0, 64), (0, 256), (0, 1024), (1, 64), (1, 256), (1, 512)} | {(b, "parts", s) for b in (0, 1) for s in (False, True)}
    assert sides == {(b, s) for b in (0, 1) for s in (False, True)}


def test_host_checks():
    from maloq_amd import _lib
    one = 16
    for name, args, what in (
            ("maloq_group_norm_fwd", (3, one, 8, one, one, 0, 1, 1, 8, 1, 1e-5, one, one, one, None), "dtype"),
            ("maloq_group_norm_fwd", (1, one, 8, one, one, 4, 1, 1, 8, 1, 1e-5, one, one, one, None), "activation"),
            ("maloq_group_norm_fwd", (1, one, 8, one, one, 0, 1, 1, 8, 3, 1e-5, one, one, one, None), "groups"),
            ("maloq_group_norm_fwd", (1, one, 8, one, one, 0, -1, 1, 8, 1, 1e-5, one, one, one, None), "out of range"),
            ("maloq_group_norm_fwd", (1, one, 8, one, one, 0, 1, 1 << 30, 8, 1, 1e-5, one, one, one, None), "out of range"),
            ("maloq_group_norm_fwd", (1, one, 8, one, one, 0, 1, 1 << 20, 8, 1, 1e-5, None, one, one, None), "workspace"),
            ("maloq_group_norm_bwd", (1, one, 8, one, 8, one, one, None, 0, 1, 4, 8, 1, one, one, one, None), "statistics"),
            ("maloq_group_norm_bwd", (1, one, 8, one, 8, one, one, one, 0, 20000, 4, 8, 1, None, one, one, None), "workspace")):
        with pytest.raises(_lib.MaloqHipError, match=what):
            _lib.call(name, *args)
    assert _lib.load().maloq_group_norm_workspace_floats(1, 1, 1, 8, 3, 0) == -1
