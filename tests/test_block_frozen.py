"""What ``autograd.linear`` keeps for its backward pass (CPU: the kernels' functions are replaced by torch's)."""
from importlib import import_module

import pytest
import torch

BF = torch.bfloat16
NAMES = ("x", "weight", "bias", "gate", "residual")


@pytest.fixture
def ad(pkg, monkeypatch):
    ops, ad = import_module(pkg.__name__ + ".ops"), import_module(pkg.__name__ + ".autograd")

    def linear_fwd(x, weight, bias=None, activation=None, gate=None, residual=None, out_dtype=None, dropout=0.0, state=None,
                   keep=False):
        z = x @ weight.t() + bias
        y = (torch.nn.functional.gelu(z) if activation else z) * gate + residual
        return (y, z) if keep else y

    def linear_bwd(dy, x, weight, kept=None, activation=None, gate=None, dropout=0.0, state=None, need=None,
                   weight_dtype=None, param_dtype=None):
        slope = 1.0
        if activation:
            z = kept.detach().float().requires_grad_()
            with torch.enable_grad():
                slope = torch.autograd.grad(torch.nn.functional.gelu(z).sum(), z)[0]
        dz = (dy.float() * gate.float() * slope)
        act = None if kept is None else torch.nn.functional.gelu(kept.float()) if activation else kept.float()
        return (dz @ weight.float() if need[0] else None, dz.t() @ x.float() if need[1] else None,
                dz.sum(0) if need[2] else None, (dy.float() * act).sum(0) if need[3] else None)
    monkeypatch.setattr(ops, "linear_fwd", linear_fwd)
    monkeypatch.setattr(ops, "linear_bwd", linear_bwd)
    return ad


def leaves(wanted, master=False):
    g = torch.Generator().manual_seed(0)
    shapes = {"x": (6, 8), "weight": (10, 8), "bias": (10,), "gate": (10,), "residual": (6, 10)}
    ts = {n: torch.randn(*s, generator=g).to(torch.float32 if master and n == "weight" else BF) for n, s in shapes.items()}
    return {n: t.requires_grad_(n in wanted) for n, t in ts.items()}


@pytest.mark.parametrize("activation", [None, "gelu"])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("which", range(1, 32))
def test_only_what_a_gradient_reads_is_kept(ad, activation, master, which):
    """x for the weight's gradient, the weight (or its rounded copy) for x's, and for any set of them the gradients come out."""
    wanted = {n for j, n in enumerate(NAMES) if which >> j & 1}
    t = leaves(wanted, master)
    y = ad.linear(t["x"], t["weight"], t["bias"], activation, t["gate"], t["residual"])
    saved = [s for s in y.grad_fn.saved_tensors if s is not None]
    assert ("weight" in wanted) == any(s.shape == (6, 8) for s in saved)
    assert ("x" in wanted) == any(s.shape == (10, 8) for s in saved)
    y.float().sum().backward()
    every = leaves(set(NAMES), master)
    ad.linear(every["x"], every["weight"], every["bias"], activation, every["gate"], every["residual"]).float().sum().backward()
    for n in NAMES:
        assert (t[n].grad is not None) == (n in wanted)
        assert n not in wanted or torch.equal(t[n].grad, every[n].grad)


def test_operands_that_are_read_are_asked_for(pkg):
    ops = import_module(pkg.__name__ + ".ops")
    t = torch.zeros(4, 8, dtype=BF)
    for args in ((t, None, t), (t, t, None), (t, None, None)):
        with pytest.raises(ValueError, match="dx reads the weight, dweight reads x"):
            ops.linear_bwd(*args)
    for x, w, need in ((None, t, (True, False, True, False)), (t, None, (False, True, True, False)),
                       (None, None, (False, False, True, False))):
        with pytest.raises(ValueError, match="GPU"):
            ops.linear_bwd(t, x, w, need=need)
