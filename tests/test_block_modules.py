"""What "saf3r_block" and ``linear_kernels`` make of a model's modules: which calls the kernels stand for, with which arguments,
and which are left alone (CPU: the kernels' functions are replaced by torch's)."""
from importlib import import_module

import pytest
import torch
import torch.nn.functional as F
from torch import nn

BF = torch.bfloat16


@pytest.fixture
def mods(pkg, monkeypatch):
    """(autograd, aggregator, calls): the functions that launch kernels compute with torch and note their arguments."""
    ad, agg = import_module(pkg.__name__ + ".autograd"), import_module(pkg.__name__ + ".aggregator")
    calls = []

    def qkv_attention(qkv, patterns, frames=1, pos=None, tables=None, norm=False, weight=None, bias=None, eps=1e-5,
                      token_mask=None, scale=None):
        return qkv[..., 2 * len(patterns) * 64:]

    def layer_norm(x, weight=None, bias=None, eps=1e-5, out_dtype=None):
        return F.layer_norm(x, x.shape[-1:], weight, bias, eps)

    def linear(x, weight, bias=None, activation=None, gate=None, residual=None, out_dtype=None, dropout=0.0, state=None):
        calls.append(("linear", activation, gate is not None, None if residual is None else residual.dtype, dropout))
        y = F.linear(x.float(), weight.float(), bias.float())
        y = F.gelu(y, approximate="tanh" if activation == "gelu_tanh" else "none") if activation else y
        y = y if gate is None else y * gate.float()
        return y.to(x.dtype) if residual is None else (residual.float() + y).to(residual.dtype)

    def residual_norm(x, branch, gate=None, weight=None, bias=None, eps=1e-5, dropout=0.0, state=None):
        calls.append(("residual_norm", x.dtype, branch.dtype, gate is not None, dropout))
        h = x + (branch if gate is None else branch * gate).to(x.dtype)
        return h, layer_norm(h.to(branch.dtype), weight, bias, eps)

    def dropout(x, p, training=True, state=None):
        calls.append(("dropout", p))
        return x
    for f in (qkv_attention, layer_norm, linear, residual_norm, dropout):
        monkeypatch.setattr(ad, f.__name__, f)
    return ad, agg, calls


def block(agg, drop=0.0, dtype=BF, init=0.5):
    torch.manual_seed(0)
    b = agg.Block(64, 1, 2.0, init, drop=drop).to(dtype)
    b.frame_attention = "saf3r_block"
    return b


def test_a_block_is_its_kernels(mods):
    _, agg, calls = mods
    b = block(agg)
    x = torch.randn(2, 5, 64).to(BF)
    y = b(x)
    assert calls == [("linear", None, False, None, 0.0), ("linear", None, False, None, 0.0),
                     ("residual_norm", BF, BF, True, 0.0), ("linear", "gelu", False, None, 0.0),
                     ("linear", None, True, BF, 0.0)]
    calls.clear()
    b.frame_attention = "saf3r_train"
    ref = b(x)
    assert not calls and (y.float() - ref.float()).abs().max() < 0.05 * ref.float().abs().max()


def test_dropouts(mods):
    _, agg, calls = mods
    b = block(agg, drop=0.25)
    b(torch.randn(2, 5, 64).to(BF))
    assert [c[-1] for c in calls] == [0.0, 0.0, 0.25, 0.25, 0.25]
    calls.clear()
    b.eval()(torch.randn(2, 5, 64).to(BF))
    assert [c[-1] for c in calls] == [0.0] * 5
    assert isinstance(agg.Block(64, 1).mlp.drop, nn.Identity)


def test_no_layer_scale(mods):
    _, agg, calls = mods
    block(agg, init=None)(torch.randn(2, 5, 64).to(BF))
    assert calls[2][3] is False and calls[4][2] is False


def test_products_in_fp32_are_torchs(mods):
    """An fp32 model: the residual and its norm run through the kernels, the products do not."""
    _, agg, calls = mods
    b = block(agg, dtype=torch.float32)
    b(torch.randn(2, 5, 64))
    assert calls == [("residual_norm", torch.float32, torch.float32, True, 0.0)]


class Scale(nn.Module):
    def forward(self, x):
        return 2 * x


class OtherLinear(nn.Linear):
    def forward(self, x):
        return super().forward(x) + 1


def test_modules_that_compute_differently_are_called(mods):
    _, agg, calls = mods
    x = torch.randn(2, 5, 64).to(BF)
    b = block(agg, drop=0.5)
    b.ls1 = Scale()
    b(x)
    assert ("dropout", 0.5) in calls and not [c for c in calls if c[0] == "residual_norm"]
    for change in (lambda m: setattr(m.mlp, "act", nn.ReLU()), lambda m: setattr(m.mlp, "drop", nn.AlphaDropout(0.5)),
                   lambda m: m.mlp.register_forward_hook(lambda *a: None), lambda m: setattr(m, "ls2", Scale()),
                   lambda m: setattr(m.mlp, "fc1", OtherLinear(64, 128).to(BF)),
                   lambda m: m.mlp.fc2.register_forward_hook(lambda *a: None)):
        b = block(agg)
        change(b)
        calls.clear()
        b(x)
        assert [c[0] for c in calls] == ["linear", "linear", "residual_norm"]
    b = block(agg)
    b.attn.proj.register_forward_hook(lambda *a: None)
    calls.clear()
    b(x)
    assert [c[0] for c in calls] == ["linear", "residual_norm", "linear", "linear"]
    b = block(agg)
    b.mlp.act = nn.GELU(approximate="tanh")
    calls.clear()
    b(x)
    assert calls[3][1] == "gelu_tanh"


def test_parameters_of_two_types_are_torchs(mods):
    """A bf16 model with fp32 scales: what torch's promotion makes of it."""
    _, agg, calls = mods
    b = block(agg)
    b.ls1.gamma.data = b.ls1.gamma.data.float()
    b.ls2.gamma.data = b.ls2.gamma.data.float()
    b.norm2 = b.norm2.float()
    stream = b._residual(torch.randn(2, 5, 64).to(BF), torch.randn(2, 5, 64).to(BF), 0.0)[0]
    assert stream.dtype == torch.float32 and calls == [("residual_norm", torch.float32, BF, True, 0.0)]


def test_kinds_of_a_model(mods):
    _, agg, calls = mods
    m = agg.VGGTAggregatorModel(img_size=28, embed_dim=64, depth=1, num_heads=1, dino_depth=1, dino_dim=64, dino_heads=1,
                                frame_attention="saf3r_block", drop=0.1).to(BF)
    m(torch.rand(1, 2, 3, 28, 28).to(BF))
    assert len([c for c in calls if c[0] == "residual_norm"]) == 3
    assert [c[-1] for c in calls if c[0] == "residual_norm"] == [0.0, 0.1, 0.1]  # (the patch embedding's blocks have none)
    with pytest.raises(ValueError, match="frame attention"):
        m.aggregator.set_frame_attention("other")


def test_patched_layers(pkg, mods, monkeypatch):
    """``patch_module.linear_kernels`` reaches the layers."""
    ad, agg, calls = mods
    patch = import_module(pkg.__name__ + ".patch")
    vggt = import_module(pkg.__name__ + ".vggt")
    for on in (False, True):
        model = vggt.GlobalAttentionStack(1, 64, 1)
        patch.patch_model(model, "vggt", {"patch_module": {"type": "headsparse", "linear_kernels": on},
                                          "sparse_config": {"0": []}})
        assert model.aggregator.global_blocks[0].attn.linear_kernels is on
    lin = nn.Linear(64, 32).to(BF)
    ad.module_linear(lin, torch.randn(3, 64).to(BF))
    assert calls == [("linear", None, False, None, 0.0)]
    calls.clear()
    ad.module_linear(lin.float(), torch.randn(3, 64))
    assert not calls
    assert ad.module_dropout(nn.Dropout(0.3)) == 0.3 and ad.module_dropout(nn.Dropout(0.3).eval()) == 0.0
    assert ad.module_dropout(nn.Identity()) == 0.0 and ad.module_dropout(nn.AlphaDropout(0.1)) is None
