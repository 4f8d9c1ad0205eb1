"""The feed-forward sublayer (maloq_amd.feed_forward): the norm, the linear layers and their 8-bit forms together."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _plain(layer, x, r):
    """In 64 bits."""
    p = {k: v.detach().double().requires_grad_() for k, v in layer.named_parameters()}
    h = x if r is None else x + r
    n = h * (h.square().mean(-1, keepdim=True) + layer.eps).rsqrt() * p["norm_weight"]
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[layer.act]
    a = act(n @ p["w1"].T + p.get("b1", 0))
    return h + a @ p["w2"].T + p.get("b2", 0), p


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,width,inner,act,bias", [((7,), 96, 200, "silu", True), ((3, 50), 129, 77, "gelu", False),
                                                         ((600,), 256, 1024, "gelu", True)])
def test_layer(sizes, width, inner, act, bias, dt, device):
    """Six roundings lie between input and a gradient (norm, argument, activation, product, its gradient, the result),
    each of half a step of what it rounds; in norms, with a factor of two for the paths' sums."""
    from maloq_amd.feed_forward import FeedForward
    torch.manual_seed(1)
    layer = FeedForward(width, inner, act=act, bias=bias, device=device, dtype=dt)
    with torch.no_grad():
        for p in layer.parameters():
            p.add_(0.1 * torch.randn_like(p))
    x, r, g = (torch.randn(*sizes, width, device=device).to(dt) for _ in range(3))
    lx, lr = x.clone().requires_grad_(), r.clone().requires_grad_()
    y = layer(lx, lr)
    names = [k for k, _ in layer.named_parameters()]
    got = torch.autograd.grad(y, [lx, lr, *layer.parameters()], g)
    x64, r64 = x.double().requires_grad_(), r.double().requires_grad_()
    ref, p = _plain(layer, x64, r64)
    want = torch.autograd.grad(ref, [x64, r64, *(p[k] for k in names)], g.double())
    u = torch.finfo(dt).eps / 2 if dt != torch.float32 else 2.0 ** -19
    for a, b, name in zip((y, *got), (ref, *want), ("y", "x", "residual", *names)):
        assert a.dtype == dt and (a.double() - b).norm() <= 12 * u * b.norm(), name
    y0 = layer(x)
    assert (y0.double() - _plain(layer, x.double(), None)[0]).norm() <= 12 * u * y0.double().norm()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 20, 300])
def test_served(rows, device):
    """e4m3 operands: each number is off by 2^-4 of itself at most, evenly spread about 2^-4 / sqrt(3) / 1.4 in norm,
    twice each product (x and W), through two products: below 0.1 of the sublayer's own output."""
    from maloq_amd.feed_forward import FeedForward
    torch.manual_seed(2)
    layer = FeedForward(256, 1024, device=device, dtype=torch.bfloat16)
    served = layer.quantized()
    x, r = (torch.randn(rows, 256, device=device, dtype=torch.bfloat16) for _ in range(2))
    with torch.no_grad():
        ref, _ = _plain(layer, x.double(), r.double())
        own = (ref - x.double() - r.double()).norm()
        assert (served(x, r).double() - ref).norm() <= 0.1 * own
        assert (served(x).double() - _plain(layer, x.double(), None)[0]).norm() <= 0.1 * own
        assert torch.equal(served(x[:1], r[:1]), served(x[:1], r[:1]))


@pytest.mark.gpu
def test_example(device):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import feed_forward
    finally:
        sys.path.pop(0)
    losses, off = feed_forward.main(["--width", "256", "--inner", "512", "--rows", "512", "--steps", "10"])
    assert losses[-1] < losses[0] and all(o < 0.1 for o in off)


def test_refusals():
    from maloq_amd.feed_forward import FeedForward
    for bad in (lambda: FeedForward(8, 8, act="tanh"), lambda: FeedForward(0, 8), lambda: FeedForward(16385, 8),
                lambda: FeedForward(8, 0)):
        with pytest.raises(ValueError):
            bad()
    layer = FeedForward(8, 16)
    assert sorted(k for k, _ in layer.named_parameters()) == ["b1", "b2", "norm_weight", "w1", "w2"]
    with pytest.raises(ValueError, match="GPU"):
        layer(torch.zeros(3, 8))
    with pytest.raises(ValueError, match="too long"):
        FeedForward(8, 16385).quantized()


def test_host_checks():
    """The C entries refuse what their kernels do not take before any launch."""
    from maloq_amd import _lib
    lib = _lib.load()
    one = 16  # (no pointer is read)
    calls = [
        ("maloq_linear_fwd", (9, one, 8, one, 8, None, None, 0, 0, 4, 8, 8, None, None, one, None), "dtype"),
        ("maloq_linear_fwd", (1, one, 8, one, 8, None, None, 0, 7, 4, 8, 8, None, None, one, None), "activation"),
        ("maloq_linear_fwd", (1, one, 8, one, 8, None, None, 0, 0, -1, 8, 8, None, None, one, None), "out of range"),
        ("maloq_linear_fwd", (1, one, 8, one, 8, None, None, 0, 0, 40, 8, 1 << 25, None, None, one, None), "out of range"),
        ("maloq_linear_fwd", (1, one + 2, 64, one, 64, None, None, 0, 0, 40, 64, 64, None, None, one, None), "16 bytes"),
        ("maloq_linear_fwd", (1, one, 60, one, 64, None, None, 0, 0, 40, 64, 64, None, None, one, None), "16 bytes"),
        ("maloq_linear_fwd", (1, one, 65, one, 65, None, None, 0, 0, 40, 65, 64, None, None, one, None), "workspace"),
        ("maloq_linear_fwd", (1, one, 4096, one, 4096, None, None, 0, 0, 100, 4096, 64, None, None, one, None), "workspace"),
        ("maloq_linear_fwd", (0, one, 1 << 25, one, 64, None, None, 0, 0, 40, 64, 64, None, None, one, None), "stride"),
        ("maloq_linear_quantized", (1, one, 64, None, one, 64, None, None, None, 0, 0, 40, 64, 64, None, one, None), "scales"),
        ("maloq_linear_act_bwd", (1, one, 8, None, 2, 4, 8, one, 8, None, None, None), "given"),
        ("maloq_linear_act_bwd", (1, one, 8, None, 0, 4, 8, one, 7, None, None, None), "ld_dz"),
        ("maloq_rms_norm_fwd", (1, one, 8, None, 0, one, 4, 16385, 1e-6, None, one, None, None, None, None), "16384"),
        ("maloq_rms_norm_fwd", (1, one, 8, None, 0, one, 4, 64, 1e-6, None, None, None, one, None, None), "scales"),
        ("maloq_rms_norm_bwd", (1, one, 8, None, 0, one, 8, one, one, 4, 64, None, one, one, None), "partial"),
        ("maloq_quantize_rows", (5, one, 8, 4, 64, one, one, None), "dtype"),
    ]
    for name, args, what in calls:
        with pytest.raises(_lib.MaloqHipError, match=what):
            _lib.call(name, *args)
    assert lib.maloq_linear_workspace_bytes(1, 3, 1, 1, 1) == -1 and lib.maloq_linear_workspace_bytes(1, 0, -1, 1, 1) == -1
    assert lib.maloq_linear_workspace_bytes(1, 0, 8, 4096, 4096) == 0  # a few rows: nothing beside
    assert lib.maloq_linear_workspace_bytes(1, 0, 100, 65, 64) >= 2 * 72 * (100 + 64)
    assert lib.maloq_rms_norm_bwd_partials_floats(5, 16385) == -1
