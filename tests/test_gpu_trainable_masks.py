"""Padded clips through the functions of a training step: what padded tokens hold reaches no result and no gradient."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def mods(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return tuple(importlib.import_module(pkg.__name__ + m) for m in (".autograd", ".ops"))


@pytest.mark.parametrize("norm,rotate", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -3e38])
def test_padded_rows_of_a_qkv_buffer(mods, norm, rotate, value):
    """The gradients with anything in the padded rows are those with zeros there, bit for bit, and zero in these rows."""
    ad, ops = mods
    g = torch.Generator().manual_seed(4)
    B, F, T, H = 2, 2, 45, 3
    qkv = torch.randn(B, F * T, 3 * H * 64, generator=g).to(BF).to(DEV)
    mask = (torch.rand(B, F * T, generator=g) < 0.7).to(DEV)
    mask[1, :T] = False
    dy = torch.randn(B, F * T, H * 64, generator=g).to(BF).to(DEV)
    pos = torch.randint(0, 9, (B, F * T, 2), generator=g).to(DEV) if rotate else None
    tables = ops.rope_tables(9, 100.0, DEV) if rotate else None
    params = [(torch.rand(2, 64, generator=g) + 0.5).to(DEV), torch.randn(2, 64, generator=g).to(DEV)] if norm else []

    def step(fill):
        x = torch.where(mask[..., None], qkv, fill).to(BF).requires_grad_()
        leaves = [p.clone().requires_grad_() for p in params]
        y = ad.qkv_attention(x, [ops.DENSE, ops.ANCHOR_LOCAL, ops.ANCHOR], F, pos, tables, norm,
                             *(leaves if norm else (None, None)), token_mask=mask)
        return (y.detach(), *torch.autograd.grad(y, [x, *leaves], dy))
    want, got = step(0.0), step(value)
    for a, b in zip(got, want):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    assert not got[1][~mask].any()
