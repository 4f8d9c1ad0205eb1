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
