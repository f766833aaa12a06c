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


@pytest.mark.parametrize("shape,layout", [((2, 37, 2, 3, 64), "half"), ((1, 5, 1, 2, 48), "interleaved")])
def test_inverse_rotation_of_a_broadcast_gradient(mods, shape, layout):
    """Without a norm only the gradient is read, whatever its strides and whatever the rows hold by then."""
    ad, ops = mods
    g = torch.Generator().manual_seed(5)
    x = torch.randn(shape, generator=g).to(BF).to(DEV)
    pos = torch.randint(0, 30, (*shape[:2], 1), generator=g).to(DEV)
    tables = ops.rotary_tables(30, shape[-1], device=DEV)
    dy = torch.randn(shape[:4], generator=g).to(BF).to(DEV)[..., None].expand(shape)
    want, _, _ = ops.head_rotary_bwd(dy.contiguous(), x, pos, tables, layout)
    got, dw, db = ops.head_rotary_bwd(dy, torch.full_like(x, float("nan")), pos, tables, layout)
    assert torch.equal(got, want) and dw is None and db is None
    leaf = x.clone().requires_grad_()
    row = leaf * 1.0
    y = ad.head_rotary(row, pos, tables, layout)
    with torch.no_grad():
        row.zero_()
    y.backward(dy)
    assert torch.equal(leaf.grad, want)
