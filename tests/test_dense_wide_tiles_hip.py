"""The products on tiles of 256 x 256 (maloq_amd.dense): each operand's way of lying, contractions of whole K steps and
not, rows and columns that end inside a tile and inside a lane's eight, tiles that are whole and split.  The plan
of each case is asserted, so that none of them comes to run on other tiles unseen.

Operands are small multiples of a power of two: every sum is exact in fp32, and the result is the 64-bit one rounded once."""
import ctypes

import pytest
import torch

from test_dense_hip import E32, HALVES, TINY, _act, _inputs, _slope, _u

# product, rows, inner, outer, whole K steps, split
CASES = [
    (0, 3000, 512, 4099, True, False), (0, 3000, 520, 4099, False, False), (0, 4133, 1024, 4090, True, True),
    (0, 4133, 1032, 4090, False, True), (0, 3001, 1001, 4099, False, False), (0, 4096, 1024, 4096, True, False),
    (1, 3000, 4099, 512, True, False), (1, 3000, 4104, 520, False, False), (1, 4133, 4090, 1024, True, True),
    (1, 4133, 4090, 1032, False, True), (1, 3001, 4099, 1001, False, False), (1, 4096, 4096, 1024, True, False),
    (2, 512, 4099, 3000, True, False), (2, 520, 4104, 3000, False, False), (2, 1024, 4090, 4133, True, True),
    (2, 1032, 4090, 4133, False, True), (2, 1001, 4099, 3001, False, False), (2, 1024, 4096, 4096, True, False),
]
CASES_8 = [(3000, 1024, 4099, True, False), (3000, 1032, 4099, False, False), (4133, 2048, 4090, True, True),
           (4133, 2056, 4090, False, True), (3001, 1001, 4099, False, False), (4096, 2048, 4096, True, False)]


def _plan(dtype, product, m, k, n):
    from maloq_amd import _lib
    plan = (ctypes.c_int64 * 4)()
    _lib.call("maloq_linear_plan", dtype, product, m, k, n, ctypes.cast(plan, ctypes.c_void_p).value)
    return list(plan)


def _is_wide(dtype, product, m, k, n, whole, split):
    tile, _, tail, parts = _plan(dtype, product, m, k, n)
    inner = (k, n, m)[product]
    assert tile == 256 and (tail > 0 and parts > 1) == split and (inner % (128 if dtype == 3 else 64) == 0) == whole


@pytest.mark.parametrize("product,m,k,n,whole,split", CASES)
def test_plans(product, m, k, n, whole, split):
    """(The plan of a card with 256 CUs, also where there is none.)"""
    for dtype in (1, 2):
        _is_wide(dtype, product, m, k, n, whole, split)


def test_plans_of_eight_bits_and_others():
    from maloq_amd import _lib
    for case in CASES_8:
        _is_wide(3, 0, *case)
    assert _plan(1, 0, 16, 4096, 4096)[0] == 0 and _plan(3, 0, 17, 4096, 4096)[0] == 32 and _plan(0, 0, 16, 4096, 4096)[0] == 32
    assert all(_plan(0, p, 8192, 8192, 8192)[0] == 128 for p in range(3))
    assert _plan(1, 0, 0, 4, 4)[1:3] == [0, 0]
    for bad in ((4, 0, 1, 1, 1), (1, 3, 1, 1, 1), (3, 1, 1, 1, 1), (1, 0, -1, 1, 1)):
        with pytest.raises(_lib.MaloqHipError, match="product"):
            _plan(*bad)


def _whole_numbers(gen, device, dt, most, *shape):
    return (torch.randint(-most, most + 1, shape, generator=gen).to(device) / 8).to(dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", HALVES)
@pytest.mark.parametrize("product,m,k,n,whole,split", CASES)
def test_exact(product, m, k, n, whole, split, dt, device):
    from maloq_amd import ops
    from maloq_amd.dense import linear_act
    _is_wide(1 if dt == torch.bfloat16 else 2, product, m, k, n, whole, split)
    gen = torch.Generator().manual_seed(m + n)
    x, w, g = (_whole_numbers(gen, device, dt, 8, *s) for s in ((m, k), (n, k), (m, n)))
    if product == 0:
        b, r = _whole_numbers(gen, device, dt, 64, n), _whole_numbers(gen, device, dt, 64, m, n)
        z = x.double() @ w.double().T
        for act in ("none", "relu"):
            for bias, residual in ((b, r), (None, None)):
                want = _act(z + (b.double() if bias is not None else 0), act) + (r.double() if residual is not None else 0)
                assert torch.equal(linear_act(x, w, bias, act=act, residual=residual), want.to(dt)), (act, bias is None)
        y, kept = ops.linear_act_fwd(x, w, b, 1, r, True)
        assert torch.equal(kept, (z + b.double()).to(dt)) and torch.equal(y, (torch.relu(z + b.double()) + r.double()).to(dt))
        return
    dx, dw, _ = ops.linear_act_bwd(g, x, w, None, 0, product == 1, product == 2, False)
    if product == 1:
        assert torch.equal(dx, (g.double() @ w.double()).to(dt))
    else:
        assert torch.equal(dw, (g.double().T @ x.double()).to(dt))


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k,n,whole,split", CASES_8)
def test_eight_bits_exactly(m, k, n, whole, split, out, device):
    """Scales that are powers of two: every sum is exact."""
    from maloq_amd.dense import linear_quantized
    _is_wide(3, 0, m, k, n, whole, split)
    gen = torch.Generator().manual_seed(m + k)
    q, p = (_whole_numbers(gen, device, torch.float8_e4m3fn, 15, *s) for s in ((m, k), (n, k)))
    s, t = (torch.exp2(torch.randint(-3, 1, (c,), generator=gen).float()).to(device) for c in (m, n))
    b, r = _whole_numbers(gen, device, out, 64, n), _whole_numbers(gen, device, out, 64, m, n)
    z = (q.double() @ p.double().T) * s.double()[:, None] * t.double()
    for act in ("none", "relu"):
        for bias, residual in ((b, r), (None, None)):
            want = _act(z + (b.double() if bias is not None else 0), act) + (r.double() if residual is not None else 0)
            got = linear_quantized(q, s, p, t, bias, act=act, residual=residual, dtype=out)
            assert torch.equal(got, want.to(out)), (act, bias is None)


# activations on these tiles; bounds as in test_dense_hip
@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dt", HALVES)
@pytest.mark.parametrize("m,k,n", [(3000, 520, 4099), (4133, 1024, 4090)])
def test_activations(m, k, n, dt, act, device):
    from maloq_amd.dense import linear_act
    _is_wide(1 if dt == torch.bfloat16 else 2, 0, m, k, n, k % 64 == 0, k % 64 == 0)
    x, w, b, r, g = (t.to(device) for t in _inputs(m, k, n, dt, seed=k))
    if dt == torch.float16:  # arguments beyond the type's range: their slopes are 0 and 1
        x[5, 0], x[m - 1, k - 1], w[7, 0], w[n - 1, k - 1] = 280, 280, -250, 250
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = linear_act(*leaves, act=act, residual=r)
    gx, gw = torch.autograd.grad(y, leaves[:2], g)
    x, w, b, r, g = (t.detach().double() for t in (x, w, b, r, g))
    z = x @ w.T + b
    pre = _act(z, act)
    bz = (k + 8) * E32 * (x.abs() @ w.abs().T + b.abs())

    def check(got, ref, bound, what):
        want = ref.to(got.dtype)
        far = want.isinf()
        assert torch.equal(got[far], want[far]), what
        err, lim = (got.double() - ref)[~far].abs(), (bound + _u(dt) * ref.abs() + TINY[dt])[~far]
        assert bool((err <= lim * (1 + 1e-6)).all()), (what, (err / lim.clamp_min(1e-300)).max().item())

    check(y, pre + r, 1.13 * bz + 2.0 ** -20 * (1 + z.abs()) * pre.abs() + 2 * E32 * (pre + r).abs(), "y")
    dz = g * _slope(z, act)
    near = (z.abs() <= 64).double()
    er = g.abs() * (near * (0.8 * (_u(dt) * z.abs() + bz + TINY[dt]) + 2.0 ** -20 * (1 + z.abs())) + E32) + _u(dt) * dz.abs() + TINY[dt]
    check(gx, dz @ w, er @ w.abs() + (n + 8) * E32 * (dz.abs() @ w.abs()), "dx")
    check(gw, dz.T @ x, er.T @ x.abs() + (m + 8) * E32 * (dz.abs().T @ x.abs()), "dw")
