"""Calls that the documentation allows or refuses, of group norm and of layers that keep activations in 8 bits."""
import pickle

import pytest
import torch


def test_a_sublayer_saved_before_it_had_a_choice():
    """A whole module from a file of before `checkpoint` keeps its tensors as they are."""
    from maloq_amd.feed_forward import FeedForward
    layer = FeedForward(16, 24)
    del layer.__dict__["checkpoint"]
    assert pickle.loads(pickle.dumps(layer)).checkpoint is None
    assert pickle.loads(pickle.dumps(FeedForward(16, 24, checkpoint=torch.int8))).checkpoint is torch.int8


def test_groups_are_whole():
    """A number of groups is not rounded to one."""
    from maloq_amd.norm import group_norm
    x = torch.zeros(2, 3, 10)
    for groups in (2.5, 0.5, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="groups"):
            group_norm(x, groups)


def _calls(device):
    from maloq_amd.dense import linear_act
    from maloq_amd.norm import group_norm
    w, v = torch.randn(12, 16, device=device), torch.rand(16, device=device)
    yield lambda x: group_norm(x, 4, v, v, act="silu")
    yield lambda x: group_norm(x, 2)
    yield lambda x: linear_act(x, w, act="silu", checkpoint=torch.int8)
    yield lambda x: linear_act(x, w, checkpoint=torch.int8)


@pytest.mark.gpu
def test_transforms_are_refused(device):
    """vmap, forward mode and the other transforms of torch.func raise, also where only a parameter is transformed."""
    from maloq_amd.dense import linear_act
    from maloq_amd.norm import group_norm
    from torch.autograd import forward_ad
    x, w, v = torch.randn(5, 16, device=device), torch.randn(12, 16, device=device), torch.rand(16, device=device)
    calls = [(f, x) for f in _calls(device)]
    calls += [(lambda t: group_norm(x, 4, t, v), v), (lambda t: group_norm(x, 4, v, t), v), (lambda t: linear_act(x, t, checkpoint=torch.int8), w)]
    for f, t in calls:
        for bad in (lambda: torch.func.vmap(f)(t[None]), lambda: torch.func.jvp(f, (t,), (t,)),
                    lambda: torch.func.grad(lambda s: f(s).sum())(t), lambda: torch.func.jacrev(f)(t)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                bad()
        with forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
            f(forward_ad.make_dual(t, t))
        with forward_ad.dual_level():
            plain = f(t)
        assert torch.equal(plain, f(t))
