"""int8 products, activations kept in 8 bits and group norm at their largest and smallest: offsets beyond 2^32, sizes of zero,
inputs whose rows are one row of memory."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ROWS, WIDE = 70000, 65536  # 4.6e9 values


def _row(n, dt, device, seed=0):
    return torch.randn(1, n, generator=torch.Generator().manual_seed(seed)).to(dt).to(device)


def test_pack_beyond_32_bits(device):
    from maloq_amd.dense import pack_rows, unpack_rows
    x = _row(WIDE, torch.bfloat16, device)
    q, e = pack_rows(x.expand(ROWS, WIDE))
    one = pack_rows(x)
    for r in (0, 32767, 32768, 65535, 65536, ROWS - 1):
        assert torch.equal(q[r:r + 1], one[0]) and torch.equal(e[r:r + 1], one[1]), r
    back = unpack_rows(q, e, torch.bfloat16)
    want = unpack_rows(*one, torch.bfloat16)
    assert bool((back == want).all())


def test_kept_argument_beyond_32_bits(device):
    """Every row is one row: gradients of single rows, and of the weight that times their number."""
    from maloq_amd.dense import linear_act
    x, g = _row(8, torch.bfloat16, device), _row(WIDE, torch.bfloat16, device, 2)
    w = _row(8 * WIDE, torch.bfloat16, device, 1).view(WIDE, 8).requires_grad_()
    lx = x.expand(ROWS, 8).detach().requires_grad_()
    y = linear_act(lx, w, act="silu", checkpoint=torch.int8)
    gx, = torch.autograd.grad(y, lx, g.expand(ROWS, WIDE))
    small = x.expand(40, 8).detach().requires_grad_()
    ys = linear_act(small, w, act="silu", checkpoint=torch.int8)
    gs, = torch.autograd.grad(ys, small, g.expand(40, WIDE))
    # (other tiles add 65536 products in another order: 2^-8 of a rounding, of the rows' norm)
    for r in (0, 32768, 65535, 65536, ROWS - 1):
        assert torch.equal(y[r], ys[0]), r
        assert (gx[r].float() - gs[0].float()).norm() <= 2.0 ** -7 * gs[0].float().norm(), r


def test_int8_rows_beyond_32_bits(device):
    from maloq_amd.dense import linear_quantized, quantize_rows
    gen = torch.Generator().manual_seed(3)
    q = torch.randint(-127, 128, (1, WIDE), generator=gen, dtype=torch.int8).to(device).repeat(ROWS, 1)
    q[-1] = -q[0]
    p = torch.randint(-127, 128, (24, WIDE), generator=gen, dtype=torch.int8).to(device)
    one = lambda c: torch.ones(c, device=device)
    y = linear_quantized(q, one(ROWS), p, one(24), dtype=torch.float32)
    want = (q[0].double() @ p.double().T).float()
    assert bool((y[:-1] == want).all()) and bool((y[-1] == -want).all())
    x = _row(16384, torch.float16, device).expand(270000, 16384)
    r, s = quantize_rows(x, dtype=torch.int8)
    assert bool((r == r[:1]).all()) and bool((s == s[0]).all())


@pytest.mark.parametrize("groups", [1, 4000])
def test_group_norm_beyond_32_bits(groups, device):
    """Places that are all alike have the statistics of one, but for the fp32 sums' rounding: both samples, from the first place
    to the last.  Two bf16 results are each within half a step, 2^-8 of the value, of values that are 1e-5 apart at most: within
    2^-7 of it and 1e-5 of each other."""
    from maloq_amd.norm import group_norm
    c = 60000
    x = _row(c, torch.bfloat16, device).view(1, 1, c)
    y = group_norm(x.expand(2, 40000, c), groups, act="silu")
    one = group_norm(x, groups, act="silu").float()
    for n, p in ((0, 0), (0, 39999), (1, 0), (1, 31582), (1, 39999)):
        assert bool(((y[n, p].float() - one[0, 0]).abs() <= 2.0 ** -7 * one[0, 0].abs() + 1e-5).all()), (n, p)


def test_kept_rows_of_no_size(device):
    from maloq_amd.dense import linear_act
    for dt in (torch.bfloat16, torch.float32):
        for m, k, n in ((0, 16, 24), (5, 0, 24), (5, 16, 0), (40, 0, 40)):
            for act in ("none", "silu"):
                x, w, b = (torch.randn(*s, device=device).to(dt).requires_grad_() for s in ((m, k), (n, k), (n,)))
                y = linear_act(x, w, b, act=act, checkpoint=torch.int8)
                plain = linear_act(x, w, b, act=act)
                assert torch.equal(y, plain)
                gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
                assert gx.shape == x.shape and gw.shape == w.shape and gb.shape == b.shape
                assert not gx.any() or k and n
                assert not gw.any() or m and k


def test_two_steps_at_once(device):
    """Steps of the same leaves on two streams, and a forward whose backward comes after another's."""
    from maloq_amd.dense import linear_act
    from maloq_amd.norm import group_norm
    torch.manual_seed(0)
    x, w = torch.randn(3, 200, 64, device=device).bfloat16().requires_grad_(), torch.randn(96, 64, device=device).bfloat16().requires_grad_()
    v, b = torch.rand(64, device=device).bfloat16().requires_grad_(), torch.rand(64, device=device).bfloat16().requires_grad_()
    g = torch.randn(3, 200, 96, device=device).bfloat16()
    f = lambda t: linear_act(group_norm(t, 4, v, b, act="silu"), w, act="gelu", checkpoint=torch.int8)
    want = torch.autograd.grad(f(x), (x, w, v, b), g)
    other = (2 * x).detach().requires_grad_()
    want_other = torch.autograd.grad(f(other), (other, w, v, b), g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for s, t in zip(streams, (x, other)):
        with torch.cuda.stream(s):
            outs.append(f(t))
    got = []
    for s, t, y in reversed(list(zip(streams, (x, other), outs))):
        with torch.cuda.stream(s):
            got.append(torch.autograd.grad(y, (t, w, v, b), g))
    torch.cuda.synchronize()
    assert all(torch.equal(a, e) for a, e in zip(got[1], want)) and all(torch.equal(a, e) for a, e in zip(got[0], want_other))


@pytest.mark.parametrize("act", ["none", "silu"])
def test_kept_rows_given_back_otherwise(act, device):
    """Hooks that give back kept rows of another size or type are refused, before any of them is read."""
    from maloq_amd.dense import linear_act
    x, w = (torch.randn(*s, device=device).requires_grad_() for s in ((40, 66), (34, 66)))
    for change in (lambda t: t[:-1], lambda t: t[:0], lambda t: torch.cat([t, t]), lambda t: t.to(torch.int16)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if t.dtype == torch.uint8 else t):
            y = linear_act(x, w, act=act, checkpoint=torch.int8)
        with pytest.raises(ValueError, match="kept rows"):
            torch.autograd.grad(y, (x, w), torch.ones_like(y))
