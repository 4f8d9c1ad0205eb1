"""The residual norm (maloq_amd.norm) in float16 where x + residual passes 65504: h is infinite, y and the gradients
are those of the sum.  Bounds as in test_norm_hip; the backward starts from 256 h / sqrt(..), whose rounding is h's."""
import pytest
import torch

from test_norm_hip import E32, _check, _inputs, _reference, _u

pytestmark = pytest.mark.gpu

F16 = torch.float16


def _far(rows, n, seed):
    x, r, w, g, gh = _inputs(rows, n, F16, seed=seed)
    for row, col, v in ((0, 0, 6e4), (0, n // 2, -5e4), (rows - 1, n - 1, 65504.0), (rows // 2, n // 3, -4e4)):
        x[row, col] = r[row, col] = v
    return x, r, w, g, gh


def _bounds(x, r, w, g, gh, eps):
    h64, rstd, y64 = _reference(x, r, w, eps)
    g64, u64 = g.double(), g.double() * w.double()
    dot, dot_abs = (u64 * h64).mean(-1, keepdim=True), (u64 * h64).abs().mean(-1, keepdim=True)
    f = rstd ** 2 * dot
    dx = rstd * (u64 - h64 * f) + gh.double()
    e = _u(F16) + 48 * E32
    bx = rstd * (8 * E32 * u64.abs() + h64.abs() * (e * f.abs() + rstd ** 2 * dot_abs * e * 2)) \
        + (48 + 8) * E32 * rstd * (u64.abs() + (h64 * f).abs()) + 2 * E32 * dx.abs()
    terms = g64 * h64 * rstd
    return h64, y64, dx, bx, terms.sum(0), terms.abs().sum(0) * (e + (x.shape[0] + 8) * E32)


@pytest.mark.parametrize("rows,n", [(1, 8), (1, 4096), (19, 97), (19, 128), (7, 500), (19, 1000), (5, 2048), (19, 4096), (3, 8191),
                                    (2, 16384), (1300, 130)])
def test_sums_beyond_fp16(rows, n, device):
    from maloq_amd.norm import rms_norm
    x, r, w, g, gh = _far(rows, n, seed=n)
    lx, lr, lw = (t.to(device).requires_grad_() for t in (x, r, w))
    y, h = rms_norm(lx, lw, 1e-5, residual=lr)
    got = torch.autograd.grad((y, h), (lx, lr, lw), (g.to(device), gh.to(device)))
    h64, y64, dx, bx, dw, bw = _bounds(x, r, w, g, gh, 1e-5)
    assert (h64.abs() > 65520).any() and torch.equal(h.cpu().isinf(), h64.abs() >= 65520)
    _check(y, y64, 48 * E32 * y64.abs(), F16, "y")
    _check(got[0], dx, bx, F16, "dx")
    assert torch.equal(got[0], got[1])
    _check(got[2], dw, bw, F16, "dw")
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(rms_norm(lx, lw, 1e-5, residual=lr), (y, h)))


def test_traced_sums_beyond_fp16(device):
    """The step that torch.compile traces gives the eager call's values."""
    from maloq_amd.norm import rms_norm
    x, r, w, g, gh = (t.to(device) for t in _far(19, 130, seed=3))
    lx, lr, lw = (t.requires_grad_() for t in (x, r, w))
    step = lambda a, b, c: rms_norm(a, c, 1e-5, residual=b)
    want = torch.autograd.grad(step(lx, lr, lw), (lx, lr, lw), (g, gh))
    got = torch.autograd.grad(torch.compile(step, backend="aot_eager", fullgraph=True)(lx, lr, lw), (lx, lr, lw), (g, gh))
    assert all(t.isfinite().all() for t in want) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_operators_of_the_normed_row(device):
    from maloq_amd import ops
    for dt in (F16, torch.float32):
        x, r, w, g, _ = (t.to(device) for t in _inputs(20, 36, dt, seed=1))
        unit = ops.rms_norm_fwd(x, w, 1e-6, r, True)[3]
        for op, args in ((ops.rms_norm_fwd, (x, w, 1e-6, r, True)), (ops.rms_norm_bwd, (g, None, unit, w, torch.ones(20, device=device), True, True, True))):
            torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


def test_captured_step(device):
    """A float16 training step through norm and linear layer, rows that are padded, replayed with new inputs."""
    from maloq_amd.dense import linear_act
    from maloq_amd.norm import rms_norm
    x, r, w, g, gh = (t.to(device) for t in _far(40, 130, seed=1))
    v = (torch.randn(57, 130, device=device) / 12).half()
    leaves = [t.requires_grad_() for t in (x, r, w, v)]
    out = g[:, :57].contiguous()

    def step():
        y, h = rms_norm(leaves[0], leaves[2], 1e-5, residual=leaves[1])
        z = linear_act(y, leaves[3], act="silu")
        return (z.detach(), *torch.autograd.grad((z, h), leaves, (out, gh)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (2, 3, 4):
        fresh = _far(40, 130, seed=seed)
        with torch.no_grad():
            for t, f in zip(leaves, fresh[:3]):
                t.copy_(f)
            out.copy_(fresh[3][:, :57])
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        assert all(t.isfinite().all() for t in kept) and all(torch.equal(a, e) for a, e in zip(kept, step())), seed
