"""Linear layers of which only some inputs need a gradient: the same bits as with all of them, and no memory for what is not
read."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF, FP = torch.float32, torch.bfloat16, torch.float16
NAMES = ("x", "weight", "bias", "gate", "residual")


@pytest.fixture(scope="module")
def mods(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return [importlib.import_module(pkg.__name__ + m) for m in (".autograd", ".ops")]


@pytest.mark.parametrize("rows,k,n,dt,master,residual,act,p", [
    (40, 64, 72, BF, False, BF, "gelu", 0.0), (300, 65, 131, FP, False, F32, None, 0.1),
    (300, 128, 136, BF, True, F32, "gelu", 0.1), (1, 8, 8, BF, True, None, None, 0.0), (0, 24, 16, BF, False, None, "gelu", 0.0)])
def test_any_set_of_gradients(mods, rows, k, n, dt, master, residual, act, p):
    ad = mods[0]
    g = torch.Generator().manual_seed(rows + k)

    def rnd(*shape, kind=dt):
        return torch.randn(*shape, generator=g).to(kind).to(DEV)
    pk = F32 if master else dt
    full = {"x": rnd(rows, k), "weight": 0.1 * rnd(n, k, kind=pk), "bias": rnd(n, kind=pk), "gate": rnd(n, kind=pk),
            "residual": None if residual is None else rnd(rows, n, kind=residual)}
    dy = rnd(rows, n, kind=residual or dt)
    state = torch.tensor([5, 6], device=DEV)

    def grads(wanted, gated=True):
        t = {m: None if v is None else v.detach().requires_grad_(m in wanted) for m, v in full.items()}
        y = ad.linear(t["x"], t["weight"], t["bias"], act, t["gate"] if gated else None, t["residual"], dropout=p, state=state)
        if not y.requires_grad:
            return {}
        y.backward(dy)
        return {m: v.grad for m, v in t.items() if v is not None and v.grad is not None}
    for gated in (True, False):
        names = [m for m in NAMES if full[m] is not None and (gated or m != "gate")]
        every = grads(names, gated)
        assert sorted(every) == sorted(names)
        for which in range(1 << len(names)):
            wanted = [m for j, m in enumerate(names) if which >> j & 1]
            some = grads(wanted, gated)
            assert sorted(some) == sorted(wanted)
            for m in wanted:
                assert some[m].dtype == full[m].dtype and torch.equal(some[m], every[m]), (wanted, m)


def test_operands_that_are_not_there(mods):
    ops = mods[1]
    g = torch.Generator().manual_seed(1)
    x, w, dy, kept = (torch.randn(*s, generator=g).to(BF).to(DEV) for s in ((50, 64), (72, 64), (50, 72), (50, 72)))
    gate = torch.randn(72, generator=g).to(DEV)
    dx, dw, db, dg = ops.linear_bwd(dy, x, w, kept, "gelu", gate)
    one = ops.linear_bwd(dy, None, w, kept, "gelu", gate, need=(True, False, True, True))
    assert torch.equal(one[0], dx) and one[1] is None and torch.equal(one[2], db) and torch.equal(one[3], dg)
    one = ops.linear_bwd(dy, x, None, kept, "gelu", gate, need=(False, True, False, False), weight_dtype=F32)
    assert one[0] is one[2] is one[3] is None and one[1].dtype == F32 and torch.equal(one[1].to(BF), dw)
    one = ops.linear_bwd(dy, None, None, kept, "gelu", gate, need=(False, False, True, True))
    assert one[0] is one[1] is None and torch.equal(one[2], db) and torch.equal(one[3], dg)
    plain = ops.linear_bwd(dy.float(), None, None, need=(False, False, True, False), param_dtype=F32)[2]
    assert torch.equal(plain, ops.linear_bwd(dy.float(), x, w, need=(False, False, True, False), param_dtype=F32)[2])
    for args, text in (((dy, None, w.t()), "weight must be"), ((dy, None, w.float()), "weight must be"),
                       ((dy, None, w.to(FP)), "dy must be"), ((dy, None, w[:, :0]), "weight must be"),
                       ((dy, None, w, kept.float()), "kept must be"), ((dy, None, w, kept[1:]), "kept must be"),
                       ((dy[0, 0], None, w), "last dimension")):
        with pytest.raises(ValueError, match=text):
            ops.linear_bwd(*args, need=(True, False, False, False))
    for other in (x[1:], x.cpu(), x.float()):
        with pytest.raises(ValueError, match="x must be"):
            ops.linear_bwd(dy, other, None, need=(False, True, False, False))


@pytest.mark.parametrize("act", [None, "gelu"])
def test_memory_of_a_frozen_weight(mods, act):
    """A layer's input is not kept for its input's gradient."""
    ad = mods[0]
    x = torch.randn(4096, 1024, device=DEV, dtype=BF, requires_grad=True)
    w = torch.randn(64, 1024, device=DEV, dtype=BF) / 32
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    h = x * 2
    y = ad.linear(h, w, None, act)
    del h
    held = torch.cuda.memory_allocated() - before
    assert held <= 4 * y.numel() * y.element_size()  # (y and what an activation keeps, not 4096 x 1024)
    y.backward(torch.ones_like(y))
    assert x.grad is not None and x.grad.shape == x.shape
