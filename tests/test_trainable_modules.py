"""What the training path makes of a model's modules: the rotary tables it asks for, the modules that it computes itself
and those that it leaves alone or refuses (CPU: the kernels' functions are replaced by torch's)."""
from importlib import import_module

import pytest
import torch
import torch.nn.functional as F
from torch import nn

BF = torch.bfloat16


@pytest.fixture
def mods(pkg, monkeypatch):
    """(autograd, ops, aggregator, vggt, calls): the two functions that launch kernels return plain values and note their
    arguments."""
    ad, ops, agg, vggt = (import_module(pkg.__name__ + m) for m in (".autograd", ".ops", ".aggregator", ".vggt"))
    calls = {"attention": [], "norm": []}

    def qkv_attention(qkv, patterns, frames=1, pos=None, tables=None, norm=False, weight=None, bias=None, eps=1e-5,
                      token_mask=None, scale=None):
        calls["attention"].append({"pos": pos, "tables": tables, "norm": norm, "weight": weight, "bias": bias})
        return qkv[..., 2 * len(patterns) * 64:]

    def layer_norm(x, weight=None, bias=None, eps=1e-5, out_dtype=None):
        calls["norm"].append(x.shape)
        return F.layer_norm(x, x.shape[-1:], weight, bias, eps)
    monkeypatch.setattr(ad, "qkv_attention", qkv_attention)
    monkeypatch.setattr(ad, "layer_norm", layer_norm)
    return ad, ops, agg, vggt, calls


def test_tables_hold_every_position(mods):
    """A block that is called with few tokens of far positions (a pruned sequence) is rotated by their own angles."""
    _, ops, agg, _, calls = mods
    block = agg.Block(64, 1, qk_norm=True, rope=agg.RotaryPositionEmbedding2D(100.0))
    block.frame_attention = "saf3r_train"
    pos = torch.tensor([[[0, 0], [7, 20], [3, 2]]])
    block(torch.randn(1, 3, 64), pos=pos)
    (call,) = calls["attention"]
    cos, sin = call["tables"]
    assert cos.shape[0] > 20 and sin.shape == cos.shape
    assert torch.equal(cos[:21], ops.rope_tables(21, 100.0, "cpu")[0])


def test_tables_go_by_the_patch_grid(mods, monkeypatch):
    """Steps over different numbers of views share the tables of their grid, and read no position back."""
    _, ops, agg, _, calls = mods
    model = agg.VGGTAggregatorModel(img_size=28, embed_dim=64, depth=1, num_heads=1, dino_depth=1, dino_dim=64,
                                    dino_heads=1, frame_attention="saf3r_train")
    monkeypatch.setattr(ops, "_rope_cache", {})
    monkeypatch.setattr(torch.Tensor, "item", lambda t: pytest.fail("a read from the device"))
    for views in (1, 2, 5):
        model(torch.rand(1, views, 3, 28, 42))
    rotated = [c for c in calls["attention"] if c["tables"] is not None]
    assert len(rotated) == 6 and len(ops._rope_cache) == 1
    assert all(c["tables"][0].shape[0] == 4 and int(c["pos"].max()) == 3 for c in rotated)


class ScaledNorm(nn.LayerNorm):
    """A norm that is a LayerNorm by its class and not by what it computes."""

    def forward(self, x):
        return 2 * super().forward(x)


class Doubled:
    """A forward that belongs to an instance."""

    def __init__(self, module):
        self.module = module

    def __call__(self, x):
        return 2 * type(self.module).forward(self.module, x)


def double_weight(module, args):
    nn.init.constant_(module.weight, 2.0)


def customised(kind, dim):
    """A LayerNorm whose call gives twice LayerNorm's result."""
    norm = ScaledNorm(dim) if kind == "subclass" else nn.LayerNorm(dim)
    if kind == "hook":
        norm.register_forward_hook(lambda m, args, y: 2 * y)
    elif kind == "pre-hook":  # (as a weight that is made from others for every call)
        norm.register_forward_pre_hook(double_weight)
    elif kind == "instance":
        norm.forward = Doubled(norm)
    return norm


KINDS = ("subclass", "hook", "pre-hook", "instance")


@pytest.mark.parametrize("kind", KINDS)
def test_norms_with_a_forward_of_their_own(mods, kind):
    _, _, agg, _, calls = mods
    block = agg.Block(64, 1)
    block.norm2 = customised(kind, 64)
    x = torch.randn(1, 4, 64)
    with torch.no_grad():
        block.frame_attention = "saf3r_train"
        h = block._norm(block.norm1, x)
        assert len(calls["norm"]) == 1 and torch.equal(h, F.layer_norm(x, (64,)))
        assert torch.equal(block._norm(block.norm2, x), 2 * h) and len(calls["norm"]) == 1
        block.norm1 = nn.LayerNorm((4, 64))  # over two dimensions
        assert torch.equal(block._norm(block.norm1, x), F.layer_norm(x, (4, 64))) and len(calls["norm"]) == 1


@pytest.mark.parametrize("kind", ["subclass", "hook"])
def test_attentions_with_a_forward_of_their_own(mods, kind):
    _, _, agg, vggt, calls = mods
    block = agg.Block(64, 1)
    block.frame_attention = "saf3r_train"
    seen = []
    if kind == "subclass":
        class Marked(vggt.Attention):
            def forward(self, x, pos=None):
                seen.append(1)
                return super().forward(x, pos)
        block.attn.__class__ = Marked
    else:
        block.attn.register_forward_hook(lambda m, args, y: seen.append(1))
    block(torch.randn(1, 4, 64))
    assert seen and not calls["attention"]


@pytest.mark.parametrize("name", ["q_norm", "k_norm"])
@pytest.mark.parametrize("kind", [*KINDS, "identity", "other", "eps", "weight", "bias", "shape"])
def test_head_norms_that_are_refused(mods, name, kind):
    """Norms of q and k that the kernels do not compute, or that are not alike."""
    ad, ops, _, vggt, calls = mods
    attn = vggt.Attention(128, 2, qk_norm=True)
    qkv = torch.randn(1, 4, 384).to(BF)
    ad.module_attention(attn, qkv, None, [ops.DENSE] * 2)
    (call,) = calls["attention"]
    assert call["norm"] and call["weight"].shape == (2, 64)
    setattr(attn, name, {"identity": nn.Identity, "other": lambda: nn.RMSNorm(64),
                         "eps": lambda: nn.LayerNorm(64, eps=1e-3),
                         "weight": lambda: nn.LayerNorm(64, elementwise_affine=False),
                         "bias": lambda: nn.LayerNorm(64, bias=False),
                         "shape": lambda: nn.LayerNorm((2, 64))}.get(kind, lambda: customised(kind, 64))())
    if kind == "pre-hook":
        nn.init.ones_(getattr(attn, name).weight)
    with pytest.raises(NotImplementedError, match="norm"):
        ad.module_attention(attn, qkv, None, [ops.DENSE] * 2)
    assert len(calls["attention"]) == 1


def test_head_norms_that_are_computed(mods):
    ad, ops, _, vggt, calls = mods
    qkv = torch.randn(1, 4, 384).to(BF)
    for norm, weight, bias in ((nn.Identity, False, False), (lambda: nn.LayerNorm(64), True, True),
                               (lambda: nn.LayerNorm(64, bias=False), True, False),
                               (lambda: nn.LayerNorm(64, elementwise_affine=False), False, False)):
        attn = vggt.Attention(128, 2)
        attn.q_norm, attn.k_norm = norm(), norm()
        ad.module_attention(attn, qkv, None, [ops.DENSE] * 2)
        call = calls["attention"][-1]
        assert call["norm"] == isinstance(attn.q_norm, nn.LayerNorm)
        assert (call["weight"] is not None) == weight and (call["bias"] is not None) == bias
    with pytest.raises(NotImplementedError, match="Identity and k_norm LayerNorm"):
        attn.q_norm = nn.Identity()
        ad.module_attention(attn, qkv, None, [ops.DENSE] * 2)


def test_dropout_is_refused_in_training(mods):
    """Dropout of the probabilities is no part of the kernels: refused where it would be applied, and only there."""
    ad, ops, agg, vggt, calls = mods
    qkv = torch.randn(1, 4, 384).to(BF)
    attn = vggt.Attention(128, 2, attn_drop=0.1)
    with pytest.raises(NotImplementedError, match="attn_drop 0.1"):
        ad.module_attention(attn, qkv, None, [ops.DENSE] * 2)
    attn.eval()
    ad.module_attention(attn, qkv, None, [ops.DENSE] * 2)
    attn.train()
    attn.attn_drop.p = 0.0
    ad.module_attention(attn, qkv, None, [ops.DENSE] * 2)
    del attn.attn_drop
    attn.attn_drop = 0.2  # (a plain number, as some modules keep it)
    with pytest.raises(NotImplementedError, match="attn_drop 0.2"):
        ad.module_attention(attn, qkv, None, [ops.DENSE] * 2)
    assert len(calls["attention"]) == 2


@pytest.mark.parametrize("norm", [False, True])
def test_rotary_keeps_what_its_backward_pass_reads(mods, monkeypatch, norm):
    """Without the norm the rows are not kept for the backward pass, and may change before it."""
    ad, ops, _, _, _ = mods
    read = []

    def bwd(dy, x, *args, **kw):
        read.append(x)
        return 3 * dy, None, None
    monkeypatch.setattr(ops, "head_rotary_fwd", lambda x, *args: 3 * x)
    monkeypatch.setattr(ops, "head_rotary_bwd", bwd)
    leaf = torch.randn(1, 4, 2, 3, 64, requires_grad=True)
    x = leaf * 1.0
    pos, tables = torch.zeros(1, 4, 1, dtype=torch.long), (torch.ones(1, 32), torch.zeros(1, 32))
    y = ad.head_rotary(x, pos, tables, norm=norm)
    assert (y.grad_fn.saved_tensors[0] is None) == (not norm)
    if not norm:
        with torch.no_grad():
            x.zero_()
    y.backward(torch.ones_like(y))
    assert torch.equal(leaf.grad, torch.full_like(leaf, 3.0)) and read[0].shape == leaf.shape
