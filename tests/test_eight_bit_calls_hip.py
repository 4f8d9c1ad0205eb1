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
