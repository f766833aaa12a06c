"""The gated residual with the norm behind it (``ops.residual_norm_fwd`` / ``_bwd``) and dropout (``ops.dropout``) against
the formulas in 64 bits."""
import importlib
import math

import pytest
import torch

import block_ref as R
from test_gpu_row_ops import norm_bounds

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF, FP = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-5


@pytest.fixture(scope="module")
def ops(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return importlib.import_module(pkg.__name__ + ".ops")


def close(got, want, tol, name):
    got = got.double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    err = (got - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} off, worst {float((err / tol)[bad].max()):.3g} x the bound"


def inputs(rows, dim, dt, out, seed=0, gate=True, affine=True, pdt=None):
    g = torch.Generator().manual_seed(1000 * seed + rows + 7 * dim)

    def rnd(*shape):
        return torch.randn(*shape, generator=g)
    pdt = F32 if pdt is None else pdt
    x = rnd(rows, dim) * (0.5 + 2 * torch.rand(rows, 1, generator=g)) + 0.7
    return {"x": x.to(dt), "branch": rnd(rows, dim).to(out), "gate": (0.5 * rnd(dim)).to(pdt) if gate else None,
            "weight": (1 + 0.3 * rnd(dim)).to(pdt) if affine else None, "bias": (0.2 * rnd(dim)).to(pdt) if affine else None,
            "dh": rnd(rows, dim).to(dt), "dy": rnd(rows, dim).to(out),
            "state": torch.randint(-(1 << 62), 1 << 62, (2,), generator=g)}


def double(*ts):
    return [None if t is None else t.detach().cpu().double() for t in ts]


def check(ops, i, p=0.0, put=None, with_dh=True):
    put = put or (lambda name, t: t.to(DEV))
    d = {n: None if t is None else put(n, t) for n, t in i.items()}
    rows, dim = i["x"].shape
    dt, out = i["x"].dtype, i["branch"].dtype
    factor = R.keep_factor(p, i["state"], rows, dim)
    args = dict(dropout=p, state=d["state"])
    h, y, mean, rstd = ops.residual_norm_fwd(d["x"], d["branch"], d["gate"], d["weight"], d["bias"], eps=EPS, **args)
    assert h.dtype == dt and y.dtype == out
    x, br, g, w, b, dh, dy = double(*(i[k] for k in ("x", "branch", "gate", "weight", "bias", "dh", "dy")))
    ref_h, h_tol = R.residual_norm(x, br, g, w, b, EPS, factor, dt)
    close(h, ref_h, R.rounded(ref_h, h_tol, dt), "h")
    if not with_dh:
        dh = torch.zeros_like(dh)
    ref = norm_bounds(h.double().cpu(), dy, w, b, EPS, dim)
    close(mean, ref["mean"][0], ref["mean"][1] + 1e-37, "mean")
    close(rstd, *ref["rstd"], "rstd")
    close(y, ref["y"][0], R.rounded(*ref["y"], out), "y")
    dx, dbranch, dgate, dweight, dbias = ops.residual_norm_bwd(d["dh"] if with_dh else None, d["dy"], h, mean, rstd,
                                                              d["branch"], d["gate"], d["weight"], **args)
    top = dh + ref["dx"][0]
    top_tol = ref["dx"][1] + 2 * R.E32 * top.abs()
    close(dx, top, R.rounded(top, top_tol, dt), "dx")
    gf = factor if g is None else factor * g
    close(dbranch, top * gf, R.rounded(top * gf, top_tol * gf.abs() + 3 * R.E32 * (top * gf).abs(), out), "dbranch")
    pdt = next((i[k].dtype for k in ("gate", "weight") if i[k] is not None), out)

    def summed(value, tol):
        s = value.sum(0)
        return s, R.rounded(s, tol.sum(0) + (rows + 3) * R.E32 * value.abs().sum(0), pdt)
    if g is not None:
        close(dgate, *summed(top * br * factor, top_tol * (br * factor).abs()), "dgate")
        assert dgate.dtype == pdt
    else:
        assert dgate is None
    close(dweight, *summed(*ref["dw"]), "dweight")
    close(dbias, *summed(*ref["db"]), "dbias")
    return h, y, dx, dbranch, dgate, dweight, dbias


@pytest.mark.parametrize("dt,out", [(BF, BF), (FP, FP), (F32, F32), (F32, BF), (F32, FP)])
@pytest.mark.parametrize("rows,dim", [(1, 8), (3, 64), (70, 128), (33, 200), (129, 512), (65, 1024), (17, 1536), (9, 2048),
                                      (11, 4096), (5, 8192), (41, 2), (130, 63), (19, 65), (7, 513), (9, 1027), (6, 2047),
                                      (5, 2049), (3, 8191), (1, 1)])
def test_residual_norm(ops, dt, out, rows, dim):
    check(ops, inputs(rows, dim, dt, out))


@pytest.mark.parametrize("dt,out", [(BF, BF), (F32, FP)])
@pytest.mark.parametrize("p", [0.1, 0.5, 1.0])
@pytest.mark.parametrize("rows,dim", [(70, 128), (33, 1024), (19, 1030), (7, 63)])
def test_dropped_branches(ops, dt, out, p, rows, dim):
    check(ops, inputs(rows, dim, dt, out, seed=1), p)


@pytest.mark.parametrize("gate,affine,pdt", [(False, False, None), (False, True, F32), (True, False, BF), (True, True, BF),
                                             (True, True, FP)])
def test_parameters(ops, gate, affine, pdt):
    check(ops, inputs(50, 96, BF, BF, 2, gate, affine, pdt))
    check(ops, inputs(700, 33, F32, F32, 3, gate, affine, pdt), 0.1)


def test_many_rows(ops):
    """More rows than one step of every work-group."""
    check(ops, inputs(30011, 64, BF, BF, 4))
    check(ops, inputs(9001, 129, F32, BF, 5), 0.1)


@pytest.mark.parametrize("rows,dim", [(20, 64), (9, 1027), (5, 2048)])
def test_infinities_in_dropped_places(ops, rows, dim):
    """What a dropped element of the branch holds reaches neither a result nor a gradient."""
    i = inputs(rows, dim, F32, BF, 11)
    dropped = R.keep_factor(0.5, i["state"], rows, dim) == 0
    d = {n: t.to(DEV) for n, t in i.items()}
    res = []
    for value in (1.0, math.inf, -math.inf, math.nan):
        branch = torch.where(dropped, torch.tensor(value, dtype=BF), i["branch"]).to(DEV)
        h, y, mean, rstd = ops.residual_norm_fwd(d["x"], branch, d["gate"], d["weight"], d["bias"], dropout=0.5,
                                                 state=d["state"])
        res.append((h, y, *ops.residual_norm_bwd(d["dh"], d["dy"], h, mean, rstd, branch, d["gate"], d["weight"], 0.5,
                                                 d["state"])))
    for other in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(res[0], other))


def test_without_a_gradient_of_the_stream(ops):
    check(ops, inputs(50, 96, F32, BF, 6), with_dh=False)


def test_layouts(ops):
    i = inputs(48, 104, F32, BF, 7)

    def wide(name, t):
        if t.dim() < 2:
            return t.to(DEV)
        buf = torch.full((t.shape[0], t.shape[1] + 24), float("nan"), dtype=t.dtype, device=DEV)
        buf[:, 8:8 + t.shape[1]] = t.to(DEV)
        return buf[:, 8:8 + t.shape[1]]

    def odd(name, t):
        if t.dtype == torch.int64:
            return t.to(DEV)
        buf = torch.full((t.numel() + 1,), float("nan"), dtype=t.dtype, device=DEV)
        buf[1:] = t.to(DEV).flatten()
        return buf[1:].view(t.shape)

    def turned(name, t):
        return t.t().contiguous().to(DEV).t() if t.dim() == 2 else t.to(DEV)
    want = check(ops, i, 0.1)
    for put in (wide, odd, turned):
        got = check(ops, i, 0.1, put=put)
        assert torch.equal(got[0], want[0])
    d = {n: t.to(DEV) for n, t in i.items()}
    h, y, _, _ = ops.residual_norm_fwd(d["x"].view(4, 3, 4, 104), d["branch"].view(4, 3, 4, 104), d["gate"], d["weight"],
                                       d["bias"], EPS, dropout=0.1, state=d["state"])
    assert torch.equal(h.view(48, 104), want[0]) and torch.equal(y.view(48, 104), want[1])


def test_as_the_norm_alone(ops):
    """The norm of the stream that comes out is layer_norm's."""
    i = inputs(300, 1024, BF, BF, 8)
    d = {n: t.to(DEV) for n, t in i.items()}
    h, y, mean, rstd = ops.residual_norm_fwd(d["x"], d["branch"], d["gate"], d["weight"], d["bias"])
    y2, mean2, rstd2 = ops.layer_norm_fwd(h, d["weight"], d["bias"])
    assert torch.equal(y, y2) and torch.equal(mean, mean2) and torch.equal(rstd, rstd2)


def test_no_rows_and_what_is_needed(ops):
    x = torch.zeros(0, 24, dtype=BF, device=DEV)
    one = torch.ones(24, device=DEV)
    h, y, mean, rstd = ops.residual_norm_fwd(x, x, one, one, one)
    grads = ops.residual_norm_bwd(h, y, h, mean, rstd, x, one, one)
    assert h.shape == y.shape == grads[0].shape == grads[1].shape == (0, 24)
    assert all((t == 0).all() and t.shape == (24,) for t in grads[2:])
    i = inputs(70, 72, F32, BF, 9)
    d = {n: t.to(DEV) for n, t in i.items()}
    h, y, mean, rstd = ops.residual_norm_fwd(d["x"], d["branch"], d["gate"], d["weight"], d["bias"])
    args = (d["dh"], d["dy"], h, mean, rstd, d["branch"], d["gate"], d["weight"])
    every = ops.residual_norm_bwd(*args)
    for which in range(16):
        need = tuple(bool(which >> j & 1) for j in range(4))
        some = ops.residual_norm_bwd(*args, need=need)
        assert torch.equal(some[0], every[0])
        for n, a, b in zip(need, some[1:], every[1:]):
            assert (a is not None) == n and (not n or torch.equal(a, b))


@pytest.mark.parametrize("dt", [F32, BF, FP])
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 8), (5, 63), (70, 128), (1041, 1024), (3, 8200), (4099, 9)])
@pytest.mark.parametrize("p", [0.1, 0.5, 1.0])
def test_dropout(ops, dt, rows, dim, p):
    i = inputs(rows, dim, dt, dt, 10)
    factor = R.keep_factor(p, i["state"], rows, dim)
    y = ops.dropout(i["x"].to(DEV), p, i["state"].to(DEV))
    assert y.dtype == dt
    want = i["x"].double() * factor
    assert torch.equal(y.cpu() == 0, want == 0)
    close(y, want, R.rounded(want, 2 * R.E32 * want.abs(), dt), "y")


def test_dropout_layouts(ops):
    x = torch.randn(40, 3, 50).to(BF)
    s = torch.tensor([5, 6], device=DEV)
    want = ops.dropout(x.to(DEV), 0.3, s)
    assert torch.equal(ops.dropout(x.view(120, 50).to(DEV), 0.3, s).view(x.shape), want)
    assert torch.equal(ops.dropout(x.to(DEV).transpose(0, 2).contiguous().transpose(0, 2), 0.3, s), want)
    buf = torch.zeros(120, 64, dtype=BF, device=DEV)
    buf[:, 3:53] = x.view(120, 50).to(DEV)
    assert torch.equal(ops.dropout(buf[:, 3:53], 0.3, s).view(x.shape), want)
    same = ops.dropout(x.to(DEV), 0.0, s)
    assert torch.equal(same, x.to(DEV))
    assert ops.dropout(torch.zeros(0, 7, device=DEV), 0.5, s).shape == (0, 7)
    inf = torch.full((16, 64), math.inf, device=DEV)
    y = ops.dropout(inf, 0.5, s)
    assert ((y == 0) | (y == math.inf)).all() and (y == 0).any()


def test_offsets_beyond_32_bits(ops):
    """Rows of more than 2^31 elements in all: those of the far end."""
    rows, dim = 262_211, 8192
    far = torch.arange(rows - 40, rows, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(6)
    x = torch.randn(rows, dim, generator=g, device=DEV, dtype=BF)
    state = torch.tensor([9, 1], device=DEV)
    factor = ((R.keep_bits((9, 1), 40, dim, rows - 40) >= 16384).double() * (4 / 3)).to(DEV)
    y = ops.dropout(x, 0.25, state)
    want = x[far].double() * factor
    assert ((y[far].double() - want).abs() <= R.rounded(want, 2 * R.E32 * want.abs(), BF)).all()
    h, z, mean, rstd = ops.residual_norm_fwd(x, y, dropout=0.25, state=state)
    want = x[far].double() + y[far].double() * factor
    assert ((h[far].double() - want).abs() <= R.rounded(want, 4 * R.E32 * want.abs(), BF)).all()
    dx, db, *_ = ops.residual_norm_bwd(x, z, h, mean, rstd, dropout=0.25, state=state, need=(True, False, False, False))
    few = ops.residual_norm_bwd(x[far], z[far], h[far], mean[far], rstd[far], need=(True, False, False, False))
    assert torch.equal(dx[far], few[0])
    # (the branch's: of the unrounded gradient of the stream)
    want = dx[far].double() * factor
    assert ((db[far].double() - want).abs() <= R.rounded(want, 2 * R.half_step(BF) * want.abs(), BF)).all()


def test_masks_are_independent(ops):
    """Shares of kept elements, by column and between states, within five standard deviations."""
    x = torch.ones(4096, 512, device=DEV)
    a = ops.dropout(x, 0.25, torch.tensor([1, 0], device=DEV)) > 0
    b = ops.dropout(x, 0.25, torch.tensor([1, 1], device=DEV)) > 0
    c = ops.dropout(x, 0.25, torch.tensor([2, 0], device=DEV)) > 0
    n = x.numel()
    for m in (a, b, c):
        assert abs(float(m.double().mean()) - 0.75) < 5 * math.sqrt(0.1875 / n)
        assert float((m.double().mean(0) - 0.75).abs().max()) < 5.5 * math.sqrt(0.1875 / 4096)
    for u, v in ((a, b), (a, c), (b, c), (a[:-1], a[1:]), (a[:, :-1], a[:, 1:])):
        both = float((u & v).double().mean())
        assert abs(both - 0.5625) < 5 * math.sqrt(0.5625 * 0.4375 / (n - 4096))


def test_states(ops):
    torch.manual_seed(3)
    a, b = ops.dropout_state(DEV), ops.dropout_state(DEV)
    torch.manual_seed(3)
    assert torch.equal(a, ops.dropout_state(DEV)) and not torch.equal(a, b)
    x = torch.ones(64, 64, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.dropout(x, 0.5, ops.dropout_state(DEV))
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        seen.append(held.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_streams_and_graph(ops):
    i = inputs(1000, 512, F32, BF, 11)
    d = {n: t.to(DEV) for n, t in i.items()}

    def step():
        args = dict(dropout=0.1, state=d["state"])
        h, y, mean, rstd = ops.residual_norm_fwd(d["x"], d["branch"], d["gate"], d["weight"], d["bias"], **args)
        return (h, y, *ops.residual_norm_bwd(d["dh"], d["dy"], h, mean, rstd, d["branch"], d["gate"], d["weight"], **args))
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        d["x"].copy_(inputs(1000, 512, F32, BF, 20 + seed)["x"])
        d["state"].add_(1)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        assert not torch.equal(got[0], want[0])
