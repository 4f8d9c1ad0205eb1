"""Linear layers and norms whose saved tensors go through hooks: to host memory and back, copied to other strides, or
computed again.  Hooks keep values, not memory, so the gradients have the bits of a call without them."""
import pytest
import torch

from test_dense_hip import HALVES, _inputs

pytestmark = pytest.mark.gpu

SIZES = [((40,), 33, 20), ((70,), 129, 66), ((3, 20), 45, 17), ((300,), 64, 130), ((5,), 9, 3)]  # rows of whole 16 bytes and not


def _steps(lead, k, n, dt, device):
    from maloq_amd.dense import linear_act
    from maloq_amd.norm import rms_norm
    m = torch.Size(lead).numel()
    x, w, b, r, g = (t.to(device) for t in _inputs(m, k, n, dt, seed=k))
    x, r, g = (t.reshape(*lead, -1) for t in (x, r, g))
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    v = torch.rand(k, device=device).to(dt).requires_grad_()
    yield lambda: linear_act(x, w, b, act="silu", residual=r), leaves, g
    yield lambda: linear_act(x, w, b), leaves[:3], g
    yield lambda: rms_norm(x, v, residual=x.detach())[0], [x, v], x.detach()


@pytest.mark.parametrize("dt", HALVES + [torch.float32])
@pytest.mark.parametrize("lead,k,n", SIZES)
def test_hooks(lead, k, n, dt, device):
    hooks = {"host": torch.autograd.graph.save_on_cpu(),
             "copied": torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t)}
    for f, leaves, g in _steps(lead, k, n, dt, device):
        want = torch.autograd.grad(f(), leaves, g)
        for name, hook in hooks.items():
            with hook:
                y = f()
            assert all(torch.equal(a, e) for a, e in zip(torch.autograd.grad(y, leaves, g), want)), name


@pytest.mark.parametrize("lead,k,n", SIZES)
def test_checkpoint(lead, k, n, device):
    from torch.utils.checkpoint import checkpoint
    for f, leaves, g in _steps(lead, k, n, torch.bfloat16, device):
        want = torch.autograd.grad(f(), leaves, g)
        y = checkpoint(f, use_reentrant=False)
        assert all(torch.equal(a, e) for a, e in zip(torch.autograd.grad(y, leaves, g), want))


def _across(t):
    """The same values, the first dimension next to each other in memory."""
    return t if t.dim() == 0 else t.movedim(0, -1).contiguous().movedim(-1, 0)


@pytest.mark.parametrize("dt", HALVES + [torch.float32])
@pytest.mark.parametrize("lead,k,n", SIZES)
def test_hooks_that_change_the_order_in_memory(lead, k, n, dt, device):
    for f, leaves, g in _steps(lead, k, n, dt, device):
        want = torch.autograd.grad(f(), leaves, g)
        for unpack in (_across, lambda t: torch.stack([t, t], -1)[..., 0]):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                y = f()
            assert all(torch.equal(a, e) for a, e in zip(torch.autograd.grad(y, leaves, g), want))


def test_statistics_of_any_stride(device):
    """rms_norm_bwd's one number a row: a column of a matrix, and one for all rows."""
    from maloq_amd import ops
    x, _, _, g, _ = (t.to(device) for t in _inputs(50, 96, 96, torch.float32, seed=7))
    w = torch.rand(96, device=device)
    rstd = torch.rand(50, device=device) + 0.5
    for got, same in ((torch.stack([rstd, -rstd], 1)[:, 0], rstd), (rstd[:1].expand(50), rstd[:1].repeat(50))):
        assert not got.is_contiguous()
        a, b = (ops.rms_norm_bwd(g, None, x, w, r, True, True) for r in (got, same))
        assert all(torch.equal(s, t) for s, t in zip(a, b))
