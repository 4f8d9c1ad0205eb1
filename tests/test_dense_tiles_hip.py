"""Linear layers (maloq_amd.dense) at the sizes that choose between its kernels: a few rows, tiles of 32 to
256 rows, contractions that end inside a K step and not, tiles that are split; in HIP graphs and on
another stream.  Bounds as in test_dense_hip."""
import math

import pytest
import torch

from test_dense_hip import E32, HALVES, TINY, _act, _check, _inputs, _tol, _u

pytestmark = pytest.mark.gpu


# one to sixteen rows straight from memory; up to 32 and 64 on tiles of such; rows of any length and address
@pytest.mark.parametrize("dt", HALVES)
@pytest.mark.parametrize("k,n", [(8, 1), (64, 15), (65, 16), (129, 33), (1000, 130), (2048, 700), (4090, 64)])
@pytest.mark.parametrize("m", [1, 2, 5, 15, 16, 17, 31, 32, 33, 63, 64, 65])
def test_few_rows(m, k, n, dt, device):
    from maloq_amd.dense import linear_act
    x, w, b, r, _ = (t.to(device) for t in _inputs(m, k, n, dt, seed=m * k))
    act = ["none", "relu", "silu", "gelu"][(m + n) % 4]
    y = linear_act(x, w, b, act=act, residual=r)
    d = [t.double() for t in (x, w, b, r)]
    z = d[0] @ d[1].T + d[2]
    pre = _act(z, act)
    bz = (k + 8) * E32 * (d[0].abs() @ d[1].abs().T + d[2].abs())
    _check(y, pre + d[3], 1.13 * bz + 2.0 ** -20 * (1 + z.abs()) * pre.abs() + 2 * E32 * (pre + d[3]).abs(), "y")
    # rows that start anywhere give the same
    wide = torch.zeros(n + m, k + 3, device=device, dtype=dt)
    wide[:m, 1:k + 1], wide[m:, 1:k + 1] = x, w
    assert torch.equal(linear_act(wide[:m, 1:k + 1], wide[m:, 1:k + 1], b, act=act, residual=r), y)


# tiles of 256: whole K steps and not, one round of them, the last tiles split
LARGE = [(4100, 128, 3588), (4097, 64, 4095), (4224, 1000, 4096), (4133, 1024, 4096)]


@pytest.mark.parametrize("dt", HALVES)
@pytest.mark.parametrize("m,k,n", LARGE)
def test_large(m, k, n, dt, device):
    from maloq_amd.dense import linear_act
    x, w, b, r, g = (t.to(device) for t in _inputs(m, k, n, dt, seed=k))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = linear_act(x, w, b, act="gelu", residual=r)
    gx, gw, gb = torch.autograd.grad(y, leaves, g)
    x, w, b, r, g = (t.detach().double() for t in (x, w, b, r, g))
    z = x @ w.T + b
    pre = _act(z, "gelu")
    bz = (k + 8) * E32 * (x.abs() @ w.abs().T + b.abs())
    _check(y, pre + r, 1.13 * bz + 2.0 ** -20 * (1 + z.abs()) * pre.abs() + 2 * E32 * (pre + r).abs(), "y")
    slope = 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    dz = g * slope
    er = 0.8 * g.abs() * (_u(dt) * z.abs() + bz + TINY[dt]) + 2.0 ** -20 * (1 + z.abs()) * g.abs() + _u(dt) * dz.abs() + TINY[dt]
    _check(gx, dz @ w, er @ w.abs() + (n + 8) * E32 * (dz.abs() @ w.abs()), "dx")
    _check(gw, dz.T @ x, er.T @ x.abs() + (m + 8) * E32 * (dz.abs().T @ x.abs()), "dw")
    again = linear_act(*leaves, act="gelu", residual=r.to(dt))
    assert torch.equal(again, y) and all(torch.equal(a, t) for a, t in zip(torch.autograd.grad(again, leaves, g.to(dt)), (gx, gw, gb)))


@pytest.mark.parametrize("m,k,n", [(m, k, n) for m in (1, 16, 20, 50, 4133) for k, n in ((128, 40), (1000, 4096), (1024, 4095))])
def test_eight_bits_exactly(m, k, n, device):
    """Numbers of 1/8 to 15/8 in steps of 1/8, scales that are powers of two: every sum is exact."""
    from maloq_amd.dense import linear_quantized
    gen = torch.Generator().manual_seed(m + k)
    q, p = ((torch.randint(-15, 16, s, generator=gen) / 8).to(torch.float8_e4m3fn).to(device) for s in ((m, k), (n, k)))
    s, t = (torch.exp2(torch.randint(-3, 4, (c,), generator=gen).float()).to(device) for c in (m, n))
    b, r = ((torch.randint(-64, 65, c, generator=gen) / 8).to(device) for c in ((n,), (m, n)))
    y = linear_quantized(q, s, p, t, b, act="relu", residual=r, dtype=torch.float32)
    assert torch.equal(y.double(), torch.relu((q.double() @ p.double().T) * s.double()[:, None] * t.double() + b.double()) + r.double())


# the last columns end anywhere within a lane's eight and a wave's 64 or 128, in rows that end within a tile
@pytest.mark.parametrize("dt", HALVES + [torch.float32])
@pytest.mark.parametrize("m", [30, 63, 200])
@pytest.mark.parametrize("n", [1, 7, 64 + 3, 128 + 6, 192 + 1, 256 + 59, 256 + 120, 384 + 7, 512 + 61])
def test_last_columns(m, n, dt, device):
    from maloq_amd.dense import linear_act
    k = 72
    x, w, b, r, _ = (t.to(device) for t in _inputs(m, k, n, dt, seed=m + n))
    y = linear_act(x, w, b, act="silu", residual=r)
    d = [t.double() for t in (x, w, b, r)]
    z = d[0] @ d[1].T + d[2]
    pre = _act(z, "silu")
    if dt == torch.float32:  # as a whole: the products' errors, 1.1 of them through the activation, its own 2^-20
        size = (d[0].square() @ d[1].T.square()).sum().sqrt()
        assert (y - (pre + d[3])).norm() <= 1.13 * _tol(k) * size + 2.0 ** -20 * ((1 + z.abs()) * pre.abs()).norm() + 8 * E32 * y.norm()
    else:
        bz = (k + 8) * E32 * (d[0].abs() @ d[1].abs().T + d[2].abs())
        _check(y, pre + d[3], 1.13 * bz + 2.0 ** -20 * (1 + z.abs()) * pre.abs() + 2 * E32 * (pre + d[3]).abs(), "y")


# a few tiles more than CUs: one to a CU and the rest in parts
@pytest.mark.parametrize("m,k,n", [(2100, 1024, 2048), (2081, 300, 2040), (16400, 260, 250)])
def test_fp32_last_tiles_in_parts(m, k, n, device):
    from maloq_amd.dense import linear_act
    x, w, b, r, g = (t.to(device) for t in _inputs(m, k, n, torch.float32, seed=m))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = linear_act(*leaves, residual=r)
    gx, gw = torch.autograd.grad(y, leaves[:2], g, retain_graph=True)
    assert torch.equal(linear_act(*leaves, residual=r), y)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves[:2], g), (gx, gw)))
    x, w, b, r, g = (t.detach().double() for t in (x, w, b, r, g))
    size = lambda p, q: (p.square() @ q.square()).sum().sqrt()
    assert (y - (x @ w.T + b + r)).norm() <= _tol(k) * size(x, w.T) + 8 * E32 * y.norm()
    assert (gx - g @ w).norm() <= _tol(n) * size(g, w)
    assert (gw - g.T @ x).norm() <= _tol(m) * size(g.T, x)


# contractions over many rows: more parts than 16, and their sums
@pytest.mark.parametrize("m,k,n", [(20000, 40, 48), (9001, 130, 33), (36800, 128, 128)])
def test_fp32_many_rows(m, k, n, device):
    from maloq_amd.dense import linear_act
    x, w, b, _, g = (t.to(device).requires_grad_() for t in _inputs(m, k, n, torch.float32, seed=n))
    y = linear_act(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g)
    x, w, b, g = (t.detach().double() for t in (x, w, b, g))
    size = lambda p, q: (p.square() @ q.square()).sum().sqrt()
    assert (y - (x @ w.T + b)).norm() <= _tol(k) * size(x, w.T) + 8 * E32 * y.norm()
    assert (gx - g @ w).norm() <= _tol(n) * size(g, w)
    assert (gw - g.T @ x).norm() <= _tol(m) * size(g.T, x)
    assert (gb - g.sum(0)).norm() <= (m + 8) * E32 * g.abs().sum(0).norm()


def _like(got, ref):
    """The same infinities and NaNs."""
    got, ref = got.cpu(), ref.cpu()
    return (torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.isposinf(), ref.isposinf())
            and torch.equal(got.isneginf(), ref.isneginf()))


@pytest.mark.parametrize("dt", HALVES + [torch.float32])
def test_gradients_that_are_not_finite(dt, device):
    from maloq_amd.dense import linear_act
    x, w, _, _, g = (t.to(device) for t in _inputs(300, 160, 130, dt, seed=8))
    g[3, 5], g[299, 129], g[7, 0] = float("inf"), float("nan"), -float("inf")
    x[200, 159], w[0, 1] = -float("inf"), float("inf")
    lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(linear_act(lx, lw), (lx, lw), g)
    assert _like(gx, g.cpu().double() @ w.cpu().double()) and _like(gw, g.cpu().double().T @ x.cpu().double())


@pytest.mark.parametrize("dt", HALVES)
def test_extreme_arguments(dt, device):
    """Activations far out: no overflow of their exponentials, infinity stays, NaN stays."""
    from maloq_amd.dense import linear_act
    v = torch.tensor([0.0, -0.0, 1e-7, -1e-7, 5.0, -5.0, 12.0, -12.0, 40.0, -40.0, 300.0, -300.0, 6e4, -6e4, float("inf"),
                      float("nan")], dtype=torch.float64).to(dt).to(device)
    one = torch.ones(1, 1, device=device, dtype=dt)
    for act in ("relu", "silu", "gelu"):
        for rows in (1, 40):  # a few rows; tiles
            x = v[:, None].expand(16, 1).repeat(rows, 1).contiguous().requires_grad_()
            y = linear_act(x, one, act=act)
            ref = _act(v.double(), act).to(dt)
            assert torch.equal(y.isnan()[:16, 0], ref.isnan()) and torch.equal(y.isinf()[:16, 0], ref.isinf()), act
            fine = ~(ref.isnan() | ref.isinf())
            assert bool(((y[:16, 0] - ref)[fine].abs() <= 2 * torch.finfo(dt).eps * ref[fine].abs() + 1e-6).all()), act
            gx, = torch.autograd.grad(y, x, torch.ones_like(y))
            z = v.double()[:14].requires_grad_()
            slope, = torch.autograd.grad(_act(z, act).sum(), z)
            assert bool(((gx[:14, 0] - slope).abs() <= 4 * torch.finfo(dt).eps).all()), act


def test_graph(device):
    """Captured calls replay with new inputs: a few rows, tiles with split ends, the 8-bit chain, a training step."""
    from maloq_amd.dense import linear_act, linear_quantized, quantize_rows
    from maloq_amd.norm import rms_norm, rms_norm_quantized
    dt = torch.bfloat16
    shapes = [(4, 256, 640), (50, 1000, 333), (777, 512, 640)]
    for m, k, n in shapes:
        x, w, b, r, g = (t.to(device) for t in _inputs(m, k, n, dt, seed=1))
        nw = torch.rand(k, device=device).to(dt)
        wq, ws = quantize_rows(w)
        leaves = [t.clone().requires_grad_() for t in (x, w, nw)]

        def work():
            h = rms_norm(leaves[0], leaves[2])
            y = linear_act(h, leaves[1], b, act="gelu", residual=r)
            grads = torch.autograd.grad(y, leaves, g)
            with torch.no_grad():
                q, s, hq = rms_norm_quantized(leaves[0], leaves[2], residual=leaves[0])
                return (y.detach(), *grads, linear_act(leaves[0], leaves[1], b, act="silu"), hq,
                        linear_quantized(q, s, wq, ws, b, act="silu", residual=r))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                work()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work()
        for seed in (2, 3, 4):
            fresh = _inputs(m, k, n, dt, seed=seed)
            with torch.no_grad():
                for t, f in zip((leaves[0], leaves[1]), fresh):
                    t.copy_(f)
            b.copy_(fresh[2])
            r.copy_(fresh[3])
            graph.replay()
            torch.cuda.synchronize()
            kept = [t.clone() for t in out]
            assert all(torch.equal(a, e) for a, e in zip(kept, work())), (m, k, n, seed)


def test_other_stream(device):
    from maloq_amd.dense import linear_act
    x, w, b, r, g = (t.to(device) for t in _inputs(500, 384, 640, torch.bfloat16, seed=6))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = linear_act(*leaves, act="silu", residual=r)
    want = torch.autograd.grad(y, leaves, g)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        z = linear_act(*leaves, act="silu", residual=r)
        got = torch.autograd.grad(z, leaves, g)
    side.synchronize()
    assert torch.equal(y, z) and all(torch.equal(a, e) for a, e in zip(got, want))


def test_traced(device):
    """What torch.compile's tracing sees (fake tensors) has the real calls' sizes and types."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from maloq_amd import ops
    x, w, b, r, g = (t.to(device) for t in _inputs(20, 36, 44, torch.float16, seed=2))
    q, s = ops.quantize_rows(x)
    p, t = ops.quantize_rows(w)
    y, z = ops.linear_act_fwd(x, w, b, 2, r, True)
    calls = [(ops.linear_act_fwd, (x, w, b, 2, r, True)), (ops.linear_act_bwd, (g, x, w, z, 2, True, False, True)),
             (ops.quantize_rows, (x,)), (ops.linear_quantized, (q, s, p, t, b, 1, r, torch.float16)),
             (ops.rms_norm_fwd, (x, w[0].contiguous(), 1e-6, x)), (ops.rms_norm_quantized, (x, w[0].contiguous(), 1e-6, None)),
             (ops.rms_norm_bwd, (x, None, x, w[0].contiguous(), torch.ones(20, device=device), True, True))]
    for f, args in calls:
        real = f(*args)
        with FakeTensorMode() as mode:
            fake = f(*[mode.from_tensor(a) if torch.is_tensor(a) else a for a in args])
        real, fake = ([v] if torch.is_tensor(v) else v for v in (real, fake))
        assert [(v.shape, v.dtype, v.stride()) for v in real] == [(v.shape, v.dtype, v.stride()) for v in fake], f


def test_opcheck(device):
    from maloq_amd import ops
    for m, k, n, dt in ((20, 36, 44, torch.float16), (7, 33, 9, torch.float32)):
        x, w, b, r, g = (t.to(device) for t in _inputs(m, k, n, dt, seed=2))
        v = w[0].contiguous()
        q, s = ops.quantize_rows(x)
        p, t = ops.quantize_rows(w)
        z = ops.linear_act_fwd(x, w, b, 2, r, True)[1]
        for op, args in ((ops.rms_norm_fwd, (x, v, 1e-6, x)), (ops.rms_norm_fwd, (x, v, 1e-6, None)),
                         (ops.rms_norm_bwd, (x, None, x, v, torch.ones(m, device=device), True, False)),
                         (ops.rms_norm_quantized, (x, v, 1e-6, x)), (ops.quantize_rows, (x,)),
                         (ops.linear_act_fwd, (x, w, None, 0, None, True)), (ops.linear_act_fwd, (x, w, b, 3, r, False)),
                         (ops.linear_act_bwd, (g, x, w, z, 2, True, True, True)), (ops.linear_act_bwd, (g, x, w, None, 0, False, True, False)),
                         (ops.linear_quantized, (q, s, p, t, b, 1, r, dt))):
            # (the schema test scales its arguments, which torch cannot do to 8-bit ones)
            schema = () if any(torch.is_tensor(a) and a.dtype == torch.float8_e4m3fn for a in args) else ("test_schema",)
            torch.library.opcheck(op, args, test_utils=(*schema, "test_faketensor"))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_compiled_step_has_no_graph_break(dt, device):
    from maloq_amd.feed_forward import FeedForward
    torch.manual_seed(3)
    layer = FeedForward(72, 130, act="gelu", device=device, dtype=dt)
    x, r, g = (torch.randn(40, 72, device=device).to(dt) for _ in range(3))
    lx, lr = x.clone().requires_grad_(), r.clone().requires_grad_()
    leaves = [lx, lr, *layer.parameters()]
    y = layer(lx, lr)
    want = torch.autograd.grad(y, leaves, g)
    compiled = torch.compile(layer, backend="aot_eager", fullgraph=True)
    z = compiled(lx, lr)
    got = torch.autograd.grad(z, leaves, g)
    assert torch.equal(y, z) and all(torch.equal(a, b) for a, b in zip(got, want))
