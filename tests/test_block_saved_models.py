"""Modules of a model that was saved whole before they had dropout or ``linear_kernels``: they run as they did (CPU)."""
import copy
from importlib import import_module

import torch


def test_mlp_without_dropout(pkg):
    agg = import_module(pkg.__name__ + ".aggregator")
    torch.manual_seed(0)
    new, x = agg.Mlp(16, 32), torch.randn(3, 16)
    old = copy.deepcopy(new)
    del old._modules["drop"]
    assert torch.equal(old(x), new(x)) and torch.equal(old(x), old.fc2(old.act(old.fc1(x))))


def test_wrapper_without_linear_kernels(pkg):
    wrapper = import_module(pkg.__name__ + ".patch.wrapper").BaseHeadwiseSparseAttentionWrapper
    old = wrapper.__new__(wrapper)
    torch.nn.Module.__init__(old)
    assert old.linear_kernels is False
