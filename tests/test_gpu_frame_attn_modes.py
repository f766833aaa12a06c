"""How a launch of the attention over frames shares its walks, where results show it: sums that are joined in another order
have other bits."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def ops(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return importlib.import_module(pkg.__name__ + ".ops")


def step(ops, t, patterns, frames):
    out, lse, rest = ops.frame_attn_fwd(*t[:3], patterns, frames, rest=True)
    return (out, lse, rest, *ops.frame_attn_bwd(t[3], *t[:3], out, lse, patterns, frames, rest=rest))


@pytest.mark.parametrize("clips,tokens,heads", [(3, 300, 16), (1, 400, 2), (1, 37, 1)])
def test_patterns_of_one_frame_are_one_walk(ops, clips, tokens, heads):
    """Over a single frame every pattern is the dense one: the same walk, shared the same way, with the same bits."""
    g = torch.Generator(device=DEV).manual_seed(tokens)
    t = [torch.randn(clips, tokens, heads, 64, generator=g, device=DEV).to(BF) for _ in range(4)]
    want = step(ops, t, [ops.DENSE] * heads, 1)
    for pattern in (ops.ANCHOR_LOCAL, ops.ANCHOR, ops.FRAME_LOCAL):
        for a, b in zip(step(ops, t, [pattern] * heads, 1), want):
            assert torch.equal(a, b), pattern
