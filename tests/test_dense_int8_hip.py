"""int8 rows and their product (maloq_amd.dense, maloq_amd.norm) against 64 bits.

A row's integers are the nearest ones to 127 x / m, all of them: the quotient's 64-bit rounding cannot cross a half, which 127 x
(31 bits) and m (24) are at least 2^-56 of it away from unless they meet it.  A product's sum is exact; then four fp32
operations (the sum's conversion, two scales, the bias) of 2^-24 each, the activation and one rounding of the result.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
E32 = 2.0 ** -24
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
ACTS = ["none", "relu", "silu", "gelu"]
# single values and rows, edges of vectors, the kernel of a few rows, tiles of 32 to 256, parts of the contraction
SIZES = [(1, 1, 1), (1, 16, 8), (1, 300, 1), (2, 7, 9), (3, 128, 40), (16, 4096, 256), (17, 70, 90), (33, 4096, 64), (64, 160, 200),
         (100, 33, 8), (128, 128, 128), (129, 130, 131), (255, 96, 257), (300, 1000, 129), (31, 2056, 520), (600, 16384, 300),
         (4100, 72, 3588), (3900, 40, 4001)]


def _act(z, act):
    return {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[act](z)


def _ints(*s, gen):
    return torch.randint(-128, 128, s, generator=gen).to(torch.int8)


def _check_rows(x, q, scale):
    v = x.double().cpu()
    m = v.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100)
    assert q.dtype == torch.int8 and torch.equal(q.cpu().double(), torch.round(127 * v / m))
    assert bool(((scale.double().cpu() - m[..., 0] / 127).abs() <= E32 * m[..., 0] / 127).all())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 97, 256, 513, 1000, 2048, 4096, 5001, 16384])
def test_rows(n, dt, device):
    from maloq_amd.dense import quantize_rows
    gen = torch.Generator().manual_seed(n)
    x = torch.randn(37, n, generator=gen)
    x[1] = 0
    x[2] *= 2.0 ** -12
    x[3, :] = torch.randint(-254, 255, (n,), generator=gen) / 2  # halves
    x[3, 0] = 127
    x[4] = torch.randint(-9, 10, (n,), generator=gen).float()
    x = x.to(dt)
    if dt != torch.float16:
        x[5] *= 2.0 ** 125  # 127 x passes the range
        x[5].clamp_(-torch.finfo(dt).max, torch.finfo(dt).max)
        x[6] *= 2.0 ** -105  # less than the least scale
        x[7] *= 2.0 ** -90
    q, scale = quantize_rows(x.to(device), dtype=torch.int8)
    _check_rows(x, q, scale)
    wide = torch.cat([x, x], 1).to(device)
    for view in (wide[:, n:], wide[::2, :n], x[:1].to(device).expand(5, n)):
        _check_rows(view, *quantize_rows(view, dtype=torch.int8))


def test_rows_not_finite(device):
    from maloq_amd.dense import quantize_rows
    x = torch.randn(4, 300, device=device)
    x[1, 3], x[2, 299], x[3, 7] = float("inf"), float("nan"), -float("inf")
    q, scale = quantize_rows(x, dtype=torch.int8)
    assert scale.isnan().tolist() == [False, True, True, True]
    _check_rows(x[:1], q[:1], scale[:1])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [1, 97, 128, 1024, 4095, 8192, 16384])
def test_norm(n, dt, device):
    """The norm's rows: within half a step and the fp32 rounding (48 steps, test_norm_hip.py) of the 64-bit ones."""
    from maloq_amd.norm import rms_norm, rms_norm_quantized
    gen = torch.Generator().manual_seed(n)
    x, r = (torch.randn(19, n, generator=gen).to(dt).to(device) for _ in range(2))
    w = (1 + 0.2 * torch.randn(n, generator=gen)).to(dt).to(device)
    for residual in (None, r):
        got = rms_norm_quantized(x, w, 1e-6, residual=residual, dtype=torch.int8)
        h = x.double() + (0 if residual is None else r.double())
        y = h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.double()
        step = y.abs().amax(-1, keepdim=True) / 127
        assert bool(((got[1].double() - step[:, 0]).abs() <= 60 * E32 * step[:, 0]).all())
        assert bool(((got[0].double() * step - y).abs() <= (0.5 + 127 * 60 * E32) * step).all())
        if residual is not None:
            assert torch.equal(got[2], rms_norm(x, w, 1e-6, residual=r)[1])


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_product(m, k, n, out, device):
    from maloq_amd.dense import linear_quantized
    gen = torch.Generator().manual_seed(m + k)
    q, p = _ints(m, k, gen=gen).to(device), _ints(n, k, gen=gen).to(device)
    s, t = ((0.5 + torch.rand(c, generator=gen)).to(device) / 100 / k ** 0.25 for c in (m, n))
    b, r = (torch.randn(*c, generator=gen).to(out).to(device) for c in ((n,), (m, n)))
    act = ACTS[(m + n) % 4]
    y = linear_quantized(q, s, p, t, b if k % 3 else None, act=act, residual=r if m % 2 else None, dtype=out)
    z = (q.double() @ p.double().T) * s.double()[:, None] * t.double()
    ez = 4 * E32 * z.abs()
    if k % 3:
        z, ez = z + b.double(), ez + E32 * (z.abs() + b.double().abs())
    pre = _act(z, act)
    ref, bound = pre, 1.13 * ez + 2.0 ** -20 * (1 + z.abs()) * pre.abs()
    if m % 2:
        ref = pre + r.double()
    bound = bound + 2 * E32 * (pre.abs() + ref.abs()) + torch.finfo(out).eps / 2 * ref.abs() + TINY[out]
    assert bool(((y.double() - ref).abs() <= bound * (1 + 1e-6)).all())


@pytest.mark.parametrize("m,k,n", SIZES)
def test_product_exactly(m, k, n, device):
    """Scales that are powers of two: the sum, rounded to 24 bits once."""
    from maloq_amd.dense import linear_quantized
    gen = torch.Generator().manual_seed(n)
    q, p = _ints(m, k, gen=gen).to(device), _ints(n, k, gen=gen).to(device)
    s, t = (torch.exp2(torch.randint(-3, 4, (c,), generator=gen).float()).to(device) for c in (m, n))
    y = linear_quantized(q, s, p, t, dtype=torch.float32)
    assert torch.equal(y, ((q.double() @ p.double().T) * s.double()[:, None] * t.double()).float())


@pytest.mark.parametrize("m", [1, 20, 200])
def test_largest_sums(m, device):
    from maloq_amd.dense import linear_quantized
    k = 131071
    one = lambda c: torch.ones(c, device=device)
    for a, b in ((-128, -128), (-128, 127), (127, 127)):
        q, p = torch.full((m, k), a, dtype=torch.int8, device=device), torch.full((130, k), b, dtype=torch.int8, device=device)
        y = linear_quantized(q, one(m), p, one(130), dtype=torch.float32)
        assert bool((y == torch.tensor(float(a * b * k), dtype=torch.float64).float().item()).all())


def test_strides(device):
    from maloq_amd.dense import linear_quantized
    gen = torch.Generator().manual_seed(1)
    base, wide = _ints(6, 10, 80, gen=gen).to(device), _ints(48, 96, gen=gen).to(device)
    one = lambda c: torch.ones(c, device=device)
    for x, w in ((base[..., 3:67], wide[:, 5:69]), (base[..., 16:], wide[:, 16:80]), (base[:, ::2, :64], wide[::2, :64]),
                 (base[:1, :1, :64].expand(6, 10, 64), wide[:1, :64].expand(48, 64)), (base[0, 0, :64], wide[:, :64]),
                 (base[..., :64].transpose(0, 1), wide[:, :64].t().contiguous().t())):
        s = one(x[..., 0].numel()).view(x.shape[:-1])
        y = linear_quantized(x, s, w, one(w.shape[0]), dtype=torch.float32)
        assert y.shape == (*x.shape[:-1], w.shape[0]) and torch.equal(y.double(), x.double() @ w.double().T)


def test_empty(device):
    from maloq_amd.dense import linear_quantized, quantize_rows
    q, s = quantize_rows(torch.randn(0, 32, device=device), dtype=torch.int8)
    p, t = quantize_rows(torch.randn(8, 32, device=device), dtype=torch.int8)
    assert linear_quantized(q, s, p, t).shape == (0, 8)
    for m in (3, 40):
        b = torch.randn(24, device=device)
        z = lambda c: torch.zeros(c, 0, dtype=torch.int8, device=device)
        y = linear_quantized(z(m), torch.ones(m, device=device), z(24), torch.ones(24, device=device), b, act="relu", dtype=torch.float32)
        assert torch.equal(y, torch.relu(b).expand(m, 24))


@pytest.mark.parametrize("rows", [1, 24, 300])
def test_captured_and_on_another_stream(rows, device):
    """A serving step of norm and layer in a graph, replayed over new inputs, beside eager calls."""
    from maloq_amd.dense import linear_quantized, quantize_rows
    from maloq_amd.norm import rms_norm_quantized
    gen = torch.Generator().manual_seed(rows)
    make = lambda *s: torch.randn(*s, generator=gen).bfloat16().to(device)
    x, r, w, wn, b = make(rows, 512), make(rows, 512), make(700, 512), make(512), make(700)
    p, t = quantize_rows(w, dtype=torch.int8)

    def step():
        q, s, h = rms_norm_quantized(x, wn, residual=r, dtype=torch.int8)
        return linear_quantized(q, s, p, t, b, act="silu"), h

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        first = step()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, c) for a, c in zip(first, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for turn in range(4):
        x.copy_(make(rows, 512))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(kept, step())), turn


def test_refusals(device):
    from maloq_amd.dense import linear_quantized, quantize_rows
    from maloq_amd.norm import rms_norm_quantized
    x, w = torch.zeros(3, 64, device=device), torch.zeros(40, 64, device=device)
    (q, s), (p, t) = (quantize_rows(v, dtype=torch.int8) for v in (x, w))
    e, u = quantize_rows(w)
    long = torch.zeros(1, 131072, dtype=torch.int8, device=device)
    for bad in (lambda: quantize_rows(x, dtype=torch.uint8), lambda: rms_norm_quantized(x, x[0], dtype=torch.float16),
                lambda: linear_quantized(q, s, e, u), lambda: linear_quantized(q, s[:2], p, t), lambda: linear_quantized(q, s, p[:, :32], t),
                lambda: linear_quantized(q.to(torch.uint8), s, p, t), lambda: linear_quantized(q, s, p, t.double()),
                lambda: linear_quantized(q, s, p, t, x[0, :40]), lambda: linear_quantized(long, s[:1], long, t[:1]),
                lambda: quantize_rows(x.cpu(), dtype=torch.int8)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("dt", TYPES)
def test_feed_forward(dt, device):
    """The sublayer in int8 is its two layers on int8 rows, called one by one."""
    from maloq_amd.dense import linear_quantized, quantize_rows
    from maloq_amd.feed_forward import FeedForward
    from maloq_amd.norm import rms_norm_quantized
    torch.manual_seed(3)
    layer = FeedForward(96, 200, device=device, dtype=dt)
    x, r = (torch.randn(5, 7, 96, device=device).to(dt) for _ in range(2))
    served = layer.quantized(torch.int8)
    y = served(x, r)
    q, s, h = rms_norm_quantized(x, layer.norm_weight, layer.eps, residual=r, dtype=torch.int8)
    a = linear_quantized(q, s, *quantize_rows(layer.w1.detach(), dtype=torch.int8), layer.b1.detach(), act="silu", dtype=dt)
    z = linear_quantized(*quantize_rows(a, dtype=torch.int8), *quantize_rows(layer.w2.detach(), dtype=torch.int8), layer.b2.detach(),
                         residual=h, dtype=dt)
    assert torch.equal(y, z)
    with torch.no_grad():
        full = layer(x, r)
    # products of integer rows: each operand is off by at most 1 / 254 of its row's largest, about 1 / 80 in norm of normal numbers
    assert (y - full).float().norm() <= 0.1 * (full.float() - x.float() - r.float()).norm()
    with pytest.raises(ValueError):
        layer.quantized(torch.int32)
