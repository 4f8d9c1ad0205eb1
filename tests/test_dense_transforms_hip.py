"""Transforms for which the norm and the linear layers have no rules: they raise, and no call gives numbers without a
derivative that was asked for."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def _calls(device):
    from maloq_amd.dense import linear_act
    from maloq_amd.norm import rms_norm
    w, v = torch.randn(12, 16, device=device), torch.rand(16, device=device)
    yield lambda x: linear_act(x, w, act="silu")
    yield lambda x: rms_norm(x, v)
    yield lambda x: rms_norm(x, v, residual=x)[0]


def test_refused(device):
    x = torch.randn(5, 16, device=device)
    for f in _calls(device):
        for bad in (lambda: torch.func.vmap(f)(x[None]), lambda: torch.func.jvp(f, (x,), (x,)),
                    lambda: torch.func.grad(lambda t: f(t).sum())(x), lambda: torch.func.jacrev(f)(x)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                bad()
        with forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
            f(forward_ad.make_dual(x, x))
        assert f(x).isfinite().all()
