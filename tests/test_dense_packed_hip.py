"""Activations kept in 8 bits (maloq_amd.dense: pack_rows, unpack_rows, linear_act's checkpoint) against 64 bits.

Packing is exact arithmetic: every q and e is compared with a 64-bit restatement.  A layer's kept argument is within half a step
of the 64-bit one, beside the fp32 product's own rounding ((k + 8) 2^-24 of the terms' magnitudes).  Its gradients are those of the
values that it kept: the bounds are test_dense_hip.py's, without its rounding of the stored argument.
"""
import math

import pytest
import torch

from test_dense_hip import ACTS, E32, HALVES, LARGE, SIZES, TINY, _act, _check, _inputs, _slope, _tol, _u

TYPES = HALVES + [torch.float32]


def _pack(x):
    """The definition, on the CPU: (q, e) of float rows."""
    v = x.detach().cpu().double()
    n = v.shape[-1]
    b = torch.nn.functional.pad(v, (0, -n % 32)).unflatten(-1, (-1, 32))
    top = torch.where(b.isfinite(), b.abs(), 0.0).amax(-1)
    m, e = torch.frexp(top)  # top = m 2^e, 1/2 <= m < 1: exponent field e + 126
    field = torch.where(top == 0, 7, (e + 126 + (m >= 126.5 / 128).long()).clamp_min(7))  # (steps of 2^-126 at the least)
    q = torch.round(b * torch.exp2(133.0 - field.double())[..., None]).nan_to_num(-128, 127, -127)
    q = torch.where(b == torch.inf, 127, torch.where(b == -torch.inf, -127, q))
    return q.flatten(-2)[..., :n].to(torch.int8), field.to(torch.uint8)


def _unpack(q, e, dt=torch.float32):
    n, c = q.shape[-1], q.double()
    most = torch.finfo(dt if dt == torch.float16 else torch.bfloat16).max  # (fp32's beyond bf16's range become its largest)
    v = (c * torch.exp2(e.double() - 133).repeat_interleave(32, -1)[..., :n]).clamp(-most, most)
    v = torch.where(c.abs() == 127, c * math.inf, v)
    return torch.where(c == -128, math.nan, v)


def _rows(rows, n, dt, gen):
    x = torch.randn(rows, n, generator=gen)
    x[1] = 0
    x[2] = torch.randint(-255, 256, (n,), generator=gen) / 2.0  # halves of steps
    x[3] = torch.randint(120, 128, (n,), generator=gen).float() * torch.exp2(torch.randint(-3, 4, (n,), generator=gen).float())
    x[4, ::3] = 253.0 / 128  # the mantissa from which the step doubles
    x[5, ::2], x[5, 1::5] = math.inf, -math.inf
    x[6, n // 2] = math.nan
    x[7] = math.nan
    x[8] *= torch.exp2(torch.randint(-20, 12, (n,), generator=gen).float())
    x = x.to(dt)
    x[9] = torch.finfo(dt).max
    x[10, ::2] = -torch.finfo(dt).max
    x[11] = torch.finfo(dt).smallest_normal * torch.rand(n, generator=gen).to(dt)  # below the normal numbers
    if dt != torch.float16:
        x[12] = (torch.rand(n, generator=gen).double() * 2.0 ** -126).to(dt)
        x[13] = (torch.randn(n, generator=gen).double() * 2.0 ** -125).to(dt)
        x[14] = (torch.randn(n, generator=gen).double() * 2.0 ** 125).to(dt)
        x[15] = (torch.randn(n, generator=gen).double() * 2.0 ** -119).to(dt)
        x[16] = (torch.randn(n, generator=gen).double() * 2.0 ** -123).to(dt)
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 31, 32, 33, 40, 96, 1000, 1024, 4099])
def test_rows(n, dt, device):
    from maloq_amd.dense import pack_rows, unpack_rows
    gen = torch.Generator().manual_seed(n)
    x = _rows(21, n, dt, gen)
    q, e = pack_rows(x.to(device))
    want = _pack(x)
    assert q.shape == x.shape and e.shape == (21, (n + 31) // 32)
    assert torch.equal(q.cpu(), want[0]) and torch.equal(e.cpu(), want[1])
    back = unpack_rows(q, e, dt).cpu()
    exact = _unpack(*want, dt)
    assert back.dtype == dt and torch.equal(back.double().nan_to_num(1e300), exact.to(dt).double().nan_to_num(1e300))
    fine = x.double().isfinite() & (x.double().abs() < torch.finfo(dt).max / 2)
    assert torch.equal(back.double()[fine], exact[fine])  # no rounding to the type
    for other in TYPES:
        back = unpack_rows(q, e, other).cpu()
        assert torch.equal(back.nan_to_num(1.25), _unpack(*want, other).to(other).nan_to_num(1.25)), other


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
def test_rows_of_any_strides(dt, device):
    from maloq_amd.dense import pack_rows, unpack_rows
    gen = torch.Generator().manual_seed(4)
    base = torch.randn(6, 10, 90, generator=gen).to(dt).to(device)
    for x in (base[..., 3:70], base[:, ::2, :64], base.transpose(0, 1), base[:1, :1].expand(6, 10, 90), base[0, 0], base.permute(1, 2, 0)):
        q, e = pack_rows(x)
        assert torch.equal(q.cpu(), _pack(x)[0]) and torch.equal(e.cpu(), _pack(x)[1])
        assert torch.equal(unpack_rows(q.transpose(0, -1).contiguous().transpose(0, -1), e, dt), unpack_rows(q, e, dt))
    for sizes in ((0, 40), (4, 0), (3, 0, 5)):
        q, e = pack_rows(torch.zeros(sizes, device=device, dtype=dt))
        assert q.shape == sizes and unpack_rows(q, e, dt).shape == sizes


def _step(m, k, n, dt, act, device, seed=0, needs=(True, True, True), checkpoint=torch.int8):
    from maloq_amd.dense import linear_act
    bias, residual = (m + n) % 3 > 0, (k + n) % 2 > 0
    x, w, b, r, g = (t.to(device) for t in _inputs(m, k, n, dt, seed))
    leaves = [t.clone().requires_grad_(need) for t, need in zip((x, w, b), needs)]
    y = linear_act(leaves[0], leaves[1], leaves[2] if bias else None, act=act, residual=r if residual else None, checkpoint=checkpoint)
    wanted = [t for t, need in zip(leaves, (needs[0], needs[1], needs[2] and bias)) if need]
    return (x, w, b if bias else None, r if residual else None, g), y, torch.autograd.grad(y, wanted, g)


def _kept(x, w, b, r, act):
    from maloq_amd import ops
    return ops.linear_packed_fwd(x, w, b, ACTS.index(act), r, True)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALVES)
@pytest.mark.parametrize("m,k,n,act", [(*s, a) for s in SIZES for a in ACTS] + [(*s, a) for s in LARGE for a in ("none", "gelu")])
def test_sixteen_bits(m, k, n, act, dt, device):
    (x, w, b, r, g), y, grads = _step(m, k, n, dt, act, device, seed=m + n)
    kept = _kept(x, w, b, r, act)
    d = [None if t is None else t.double() for t in (x, w, b, r, g)]
    z = d[0] @ d[1].T + (0 if b is None else d[2])
    bz = (k + 8) * E32 * (d[0].abs() @ d[1].abs().T + (0 if b is None else d[2].abs()))
    pre = _act(z, act)
    y64 = pre + (0 if r is None else d[3])
    _check(y, y64, 1.13 * bz + 2.0 ** -20 * (1 + z.abs()) * pre.abs() + 2 * E32 * y64.abs(), "y")
    assert torch.equal(kept[0], y)
    x8, xe = (t.to(device) for t in _pack(x))
    assert torch.equal(kept[3], x8) and torch.equal(kept[4], xe)
    xk, zk = _unpack(x8, xe, dt), z
    if act != "none":
        zk = _unpack(kept[1], kept[2])
        step = torch.exp2(kept[2].double() - 133).repeat_interleave(32, -1)[:, :n]
        assert bool(((zk - z).abs() <= step * (1 if act == "relu" else 0.5) + bz).all())  # (relu: what is less than half a step is one)
        blocks = torch.nn.functional.pad(kept[1].int().abs(), (0, -n % 32)).unflatten(-1, (-1, 32)).amax(-1)
        assert bool(((blocks >= 63) & (blocks <= 126)).all())
    dz = d[4] * _slope(zk, act)
    ez = 2.0 ** -20 * (1 + zk.abs()) * d[4].abs() if act in ("silu", "gelu") else 0 * dz
    er = ez + (_u(dt) * dz.abs() + TINY[dt] if act != "none" else 0)
    _check(grads[0], dz @ d[1], er @ d[1].abs() + (n + 8) * E32 * (dz.abs() @ d[1].abs()), "dx")
    _check(grads[1], dz.T @ xk, er.T @ xk.abs() + (m + 8) * E32 * (dz.abs().T @ xk.abs()), "dw")
    if b is not None:
        _check(grads[2], dz.sum(0), ez.sum(0) + (m + 8) * E32 * dz.abs().sum(0), "db")


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,k,n", SIZES + LARGE[:1])
def test_fp32(m, k, n, act, device):
    (x, w, b, r, g), y, grads = _step(m, k, n, torch.float32, act, device, seed=m + n)
    kept = _kept(x, w, b, r, act)
    d = [None if t is None else t.double() for t in (x, w, b, r, g)]
    z = d[0] @ d[1].T + (0 if b is None else d[2])
    x8, xe = (t.to(device) for t in _pack(x))
    assert torch.equal(kept[3], x8) and torch.equal(kept[4], xe) and torch.equal(kept[0], y)
    xk, zk = _unpack(x8, xe), z
    size = lambda p, q: (p.square() @ q.square()).sum().sqrt()
    off = lambda a, t: (a.double() - t).norm()
    if act != "none":
        zk = _unpack(kept[1], kept[2])
        step = torch.exp2(kept[2].double() - 133).repeat_interleave(32, -1)[:, :n]
        near = 16 * (k + 8) * E32 * (d[0].abs() @ d[1].abs().T + 1)
        assert bool(((zk - z).abs() <= step * (1 if act == "relu" else 0.5) + near).all())
    dz = d[4] * _slope(zk, act)
    ed = 16 * E32 * ((1 + zk.abs()) * d[4]).norm() if act in ("silu", "gelu") else 0
    op = lambda t: torch.linalg.matrix_norm(t, 2)
    assert off(grads[0], dz @ d[1]) <= _tol(n) * size(dz, d[1]) + (ed + E32 * dz.norm()) * op(d[1]) + 1e-300
    assert off(grads[1], dz.T @ xk) <= _tol(m) * size(dz.T, xk) + (ed + E32 * dz.norm()) * op(xk) + 1e-300
    if b is not None:
        assert off(grads[2], dz.sum(0)) <= (m + 8) * E32 * dz.abs().sum(0).norm() + ed * math.sqrt(m)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,k,n", [(40, 64, 96), (300, 129, 66), (700, 1000, 333), (17, 4096, 64)])
def test_what_does_not_change(m, k, n, dt, device):
    """y above 16 rows; relu's slopes, whose sign is kept; a layer's dx and db without activation."""
    for act in ACTS:
        (*_, r, g), y, grads = _step(m, k, n, dt, act, device, seed=5)
        _, y0, grads0 = _step(m, k, n, dt, act, device, seed=5, checkpoint=None)
        assert torch.equal(y, y0)
        if act in ("none", "relu"):
            assert torch.equal(grads[0], grads0[0]) and all(torch.equal(a, c) for a, c in zip(grads[2:], grads0[2:])), act


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradient_against_differences(dt, act, device):
    """test_dense_hip.py's, with what the kept values are off by: dw by |dz| |x^ - x|, all three by the slope's change,
    0.8 |z^ - z| (the second derivative of gelu is at most 0.8, of silu 0.5)."""
    from maloq_amd.dense import linear_act
    x, w, b, r, c = (t.to(device) for t in _inputs(40, 56, 72, dt, seed=9))
    dirs = [torch.randn_like(t.float()) for t in (x, w, b)]

    def loss(e):
        a = [t.float() + e * d for t, d in zip((x, w, b), dirs)]
        return (linear_act(*a, act=act).double() * c.double()).sum()

    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(linear_act(*leaves, act=act, checkpoint=torch.int8), leaves, c)
    terms = [(g.double() * d.double()) for g, d in zip(got, dirs)]
    want, size = sum(t.sum() for t in terms), sum(t.abs().sum() for t in terms)
    z = x.double() @ w.double().T + b.double()
    half = lambda v: torch.exp2(_pack(v)[1].to(device).double() - 134).repeat_interleave(32, -1)[:, :v.shape[1]]
    dx, dw, db = (d.double().abs() for d in dirs)
    moved = dx @ w.double().abs().T + x.double().abs() @ dw.T + db  # the argument's change at most
    kept = (0.8 * c.double().abs() * 1.1 * half(z.float()) * moved).sum() + (1.13 * c.double().abs() * (half(x) @ dw.T)).sum()
    e = 2.0 ** -6
    assert abs((loss(e) - loss(-e)) / (2 * e) - want) <= size * (2.0 ** -9 + 3 * _u(dt)) + kept
    assert kept < 2 * size  # (a bound that says something: wrong signs or factors of two would pass it otherwise)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lead,k,n", [((40,), 64, 96), ((70,), 129, 66), ((3, 20), 45, 17), ((5,), 9, 3)])
def test_needs_hooks_and_what_is_kept(lead, k, n, dt, device):
    from maloq_amd.dense import linear_act
    m = torch.Size(lead).numel()
    x, w, b, r, g = (t.to(device) for t in _inputs(m, k, n, dt, seed=3))
    x, r, g = (t.reshape(*lead, -1) for t in (x, r, g))

    def run(needs, hooks=None, act="silu"):
        leaves = [t.clone().requires_grad_(need) for t, need in zip((x, w, b, r), needs)]
        if hooks is None:
            y = linear_act(*leaves[:3], act=act, residual=leaves[3], checkpoint=torch.int8)
        else:
            with torch.autograd.graph.saved_tensors_hooks(*hooks):
                y = linear_act(*leaves[:3], act=act, residual=leaves[3], checkpoint=torch.int8)
        return torch.autograd.grad(y, [t for t in leaves if t.requires_grad], g)

    full = run((True,) * 4)
    for bits in range(1, 15):
        needs = [bool(bits >> i & 1) for i in range(4)]
        assert all(torch.equal(a, f) for a, f in zip(run(needs), [f for f, want in zip(full, needs) if want])), needs
    for unpack in (lambda t: t.clone(), lambda t: torch.stack([t, t], -1)[..., 0], lambda t: t.to(device)):
        saved = []
        pack = lambda t: (saved.append(t), t)[1]
        assert all(torch.equal(a, f) for a, f in zip(run((True,) * 4, (pack, unpack)), full))
    kp = k + -k % (4 if dt == torch.float32 else 8)
    weights = n * kp * w.element_size()
    assert sum(t.numel() * t.element_size() for t in saved) - weights == m * (k + (k + 31) // 32 + n + (n + 31) // 32)
    for act, needs, bytes_ in (("none", (True, True, True, True), m * (k + (k + 31) // 32)), ("relu", (True, False, True, False), m * (n + (n + 31) // 32)),
                               ("none", (True, False, True, True), 0)):
        saved = []
        run(needs, (lambda t: (saved.append(t), t)[1], lambda t: t), act)
        assert sum(t.numel() * t.element_size() for t in saved) - weights == bytes_


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
def test_not_finite(dt, device):
    """Infinities and NaN in x reach the gradients that they belong to, and no others."""
    from maloq_amd.dense import linear_act
    x, w, b, r, g = (t.to(device) for t in _inputs(140, 96, 150, dt, seed=5))
    clean = _step(140, 96, 150, dt, "silu", device, seed=5)[2]
    bad = x.clone()
    bad[7, 5], bad[139, 95], bad[20, 40] = math.nan, math.inf, -math.inf
    leaves = [t.clone().requires_grad_() for t in (bad, w)]
    gx, gw = torch.autograd.grad(linear_act(*leaves, b, act="none", checkpoint=torch.int8), leaves, g)
    assert bool(gx.isfinite().all())
    cols = torch.zeros(96, dtype=torch.bool, device=device)
    cols[[5, 95, 40]] = True
    assert not gw[:, cols].isfinite().any() and bool(gw[:, ~cols].isfinite().all()) and bool(gw[:, 5].isnan().all())
    assert torch.equal(gw[:, 95].isposinf(), g[139] > 0) and torch.equal(gw[:, 40].isposinf(), g[20] < 0)
    leaves = [t.clone().requires_grad_() for t in (bad, w)]
    gx, gw = torch.autograd.grad(linear_act(*leaves, b if (140 + 150) % 3 else None, act="silu", checkpoint=torch.int8), leaves, g)
    keep = [i for i in range(140) if i not in (7, 139, 20)]
    assert torch.equal(gx[keep], clean[0][keep])


@pytest.mark.gpu
def test_infinite_arguments(device):
    """fp16 products beyond 65504: kept as they are, slopes 0 and 1."""
    from maloq_amd.dense import linear_act
    x = torch.full((40, 64), 200.0, device=device, dtype=torch.float16).requires_grad_()
    w = torch.full((64, 64), 60.0, device=device, dtype=torch.float16)
    w[::2] *= -1
    for act in ("relu", "silu", "gelu"):
        y = linear_act(x, w, act=act, checkpoint=torch.int8)
        gx, = torch.autograd.grad(y, x, torch.full_like(y, 2.0 ** -10))
        assert torch.equal(gx, torch.full_like(gx, 32 * 60 * 2.0 ** -10)), act


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,k,n", [(4, 256, 640), (50, 1000, 333), (777, 512, 640)])
def test_captured_and_on_another_stream(m, k, n, dt, device):
    from maloq_amd.dense import linear_act
    x, w, b, r, g = (t.to(device) for t in _inputs(m, k, n, dt, seed=1))
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def work():
        y = linear_act(*leaves, act="gelu", residual=r, checkpoint=torch.int8)
        return (y.detach(), *torch.autograd.grad(y, leaves, g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(first, work()))
    del first
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in (2, 3, 4):
        fresh = _inputs(m, k, n, dt, seed=seed)
        with torch.no_grad():
            for t, f in zip((x, w, b, r, g), fresh):
                t.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        assert all(torch.equal(a, c) for a, c in zip(kept, work())), seed


@pytest.mark.gpu
def test_traced(device):
    from maloq_amd import ops
    for m, k, n, dt in ((20, 36, 44, torch.float16), (7, 33, 9, torch.float32)):
        x, w, b, r, g = (t.to(device) for t in _inputs(m, k, n, dt, seed=2))
        y, z8, ze, x8, xe = ops.linear_packed_fwd(x, w, b, 2, r, True)
        for op, args in ((ops.pack_rows, (x,)), (ops.unpack_rows, (x8, xe, dt)), (ops.linear_packed_fwd, (x, w, b, 3, r, True)),
                         (ops.linear_packed_fwd, (x, w, None, 0, None, False)), (ops.linear_packed_fwd, (x, w, b, 0, None, True)),
                         (ops.linear_packed_bwd, (g, x8, xe, w, z8, ze, 2, True, True, True)),
                         (ops.linear_packed_bwd, (g, None, None, w, z8, ze, 1, True, False, True)),
                         (ops.linear_packed_bwd, (g, x8, xe, w, None, None, 0, False, True, False))):
            torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_feed_forward(dt, device):
    """The sublayer with kept activations is its layers with them; compiled, it gives the same bits."""
    from maloq_amd.dense import linear_act
    from maloq_amd.feed_forward import FeedForward
    from maloq_amd.norm import rms_norm
    torch.manual_seed(3)
    layer = FeedForward(72, 130, act="gelu", device=device, dtype=dt, checkpoint=torch.int8)
    x, r, g = (torch.randn(40, 72, device=device).to(dt) for _ in range(3))
    lx, lr = x.requires_grad_(), r.requires_grad_()
    leaves = [lx, lr, *layer.parameters()]
    got = torch.autograd.grad(layer(lx, lr), leaves, g)
    nrm, h = rms_norm(lx, layer.norm_weight, layer.eps, residual=lr)
    a = linear_act(nrm, layer.w1, layer.b1, act="gelu", checkpoint=torch.int8)
    want = torch.autograd.grad(linear_act(a, layer.w2, layer.b2, residual=h, checkpoint=torch.int8), leaves, g)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    y = torch.compile(layer, backend="aot_eager", fullgraph=True)(lx, lr)
    assert torch.equal(y, layer(lx, lr)) and all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, g), want))


@pytest.mark.gpu
def test_example(device):
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    try:
        import feed_forward
    finally:
        sys.path.pop(0)
    losses, off = feed_forward.main(["--width", "256", "--inner", "512", "--rows", "300", "--steps", "3", "--checkpoint"])
    assert len(losses) == 3 and all(math.isfinite(v) for v in losses + off)


@pytest.mark.gpu
def test_refusals(device):
    from maloq_amd import ops
    from maloq_amd.dense import linear_act, pack_rows, unpack_rows
    x, w = torch.zeros(3, 64, device=device), torch.zeros(40, 64, device=device)
    q, e = pack_rows(x)
    r = torch.zeros(3, 40, device=device)
    z = pack_rows(r)
    for bad in (lambda: linear_act(x, w, checkpoint=torch.float8_e4m3fn), lambda: pack_rows(x.double()), lambda: pack_rows(x.cpu()),
                lambda: unpack_rows(q, e[:, :1], torch.float32), lambda: unpack_rows(q, e.to(torch.int8), torch.float32),
                lambda: unpack_rows(e, q, torch.float32), lambda: unpack_rows(q, e, torch.float64), lambda: pack_rows(x.sum()),
                lambda: ops.linear_packed_bwd(r, None, None, w, *z, 2, True, True, True),
                lambda: ops.linear_packed_bwd(r, q, e, w, None, None, 2, True, True, True),
                lambda: ops.linear_packed_bwd(r[:2], q, e, w, *z, 2, True, True, True),
                lambda: ops.linear_packed_bwd(r, q, e, w, z[0], z[1][:, :1], 2, True, True, True),
                lambda: ops.linear_packed_bwd(r, q[:, :32], e[:, :1], w, *z, 2, True, True, True)):
        with pytest.raises(ValueError):
            bad()
    lx = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(linear_act(lx, w, checkpoint=torch.int8), lx, torch.ones_like(r), create_graph=True)


def test_module_refusal():
    from maloq_amd.feed_forward import FeedForward
    with pytest.raises(ValueError, match="8 bits"):
        FeedForward(8, 8, checkpoint=torch.float16)


def test_host_checks():
    """The C entries refuse what their kernels do not take before any launch."""
    from maloq_amd import _lib
    one = 16  # (no pointer is read)
    for name, args, what in (
            ("maloq_pack_rows", (3, one, 8, 4, 64, one, one, None), "dtype"),
            ("maloq_pack_rows", (1, one, 8, -1, 64, one, one, None), "out of range"),
            ("maloq_pack_rows", (1, one, 8, 4, 1 << 24, one, one, None), "out of range"),
            ("maloq_unpack_rows", (1, one, one, 4, 64, one, 63, None), "out of range"),
            ("maloq_linear_packed_fwd", (1, one, 64, one, 64, None, None, 0, 2, 40, 64, 64, None, None, one, one, None), "place"),
            ("maloq_linear_packed_fwd", (3, one, 64, one, 64, None, None, 0, 2, 40, 64, 64, None, one, one, one, None), "dtype"),
            ("maloq_linear_packed_act_bwd", (1, one, 64, None, one, 1, 40, 64, one, 64, None, None, None, None, 0, None, 0, None), "needs what"),
            ("maloq_linear_packed_act_bwd", (1, one, 64, one, None, 1, 40, 64, one, 64, None, None, None, None, 0, None, 0, None), "needs what"),
            ("maloq_linear_packed_act_bwd", (1, one, 64, one, one, 1, 40, 64, one, 64, None, None, None, one, 64, one, 64, None), "both their parts"),
            ("maloq_linear_packed_act_bwd", (1, one, 64, one, one, 1, 40, 64, one, 64, None, None, one, one, 64, one, 63, None), "out of range"),
            ("maloq_quantize_rows_int8", (5, one, 8, 4, 64, one, one, None), "dtype"),
            ("maloq_rms_norm_int8_fwd", (1, one, 8, None, 0, one, 4, 16385, 0.0, None, one, one, None), "values"),
            ("maloq_linear_int8", (1, one, 64, None, one, 64, None, None, None, 0, 0, 40, 64, 64, None, one, None), "scales"),
            ("maloq_linear_int8", (1, one, 131072, one, one, 131072, one, None, None, 0, 0, 40, 131072, 64, None, one, None), "32 bits")):
        with pytest.raises(_lib.MaloqHipError, match=what):
            _lib.call(name, *args)
    lib = _lib.load()
    assert lib.maloq_linear_packed_workspace_bytes(3, 4, 4, 4) == -1 and lib.maloq_linear_packed_workspace_bytes(1, -1, 4, 4) == -1
