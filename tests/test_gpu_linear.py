"""Linear layers with their epilogue and their gradients (``ops.linear_fwd`` / ``ops.linear_bwd``) against the formulas in 64
bits."""
import importlib
import math

import pytest
import torch

import block_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF, FP = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return importlib.import_module(pkg.__name__ + ".ops")


def close(got, want, tol, name):
    got = got.double().to(want.device)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    err = (got - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} off, worst {float((err / tol)[bad].max()):.3g} x the bound"


def inputs(rows, k, n, dt, seed=0, bias=True, gate=True, residual=None, pdt=None, ydt=None):
    g = torch.Generator().manual_seed(1000 * seed + rows + 7 * k + 13 * n)

    def rnd(*shape):
        return torch.randn(*shape, generator=g)
    pdt = dt if pdt is None else pdt
    ydt = residual if residual is not None else dt if ydt is None else ydt
    return {"x": rnd(rows, k).to(dt), "weight": (rnd(n, k) / math.sqrt(k)).to(dt),
            "bias": (0.3 * rnd(n)).to(pdt) if bias else None, "gate": (0.3 * rnd(n)).to(pdt) if gate else None,
            "residual": (2 * rnd(rows, n)).to(residual) if residual is not None else None,
            "dy": (0.1 * rnd(rows, n)).to(ydt), "state": torch.randint(-(1 << 62), 1 << 62, (2,), generator=g)}


def double(where, *ts):
    return [None if t is None else t.detach().to(where).double() for t in ts]


def check(ops, i, act=None, p=0.0, out_dtype=None, put=None, where="cpu"):
    """Forward and backward of inputs i; ``put`` moves them to the GPU in a layout of its own; the formulas on ``where``."""
    put = put or (lambda name, t: t.to(DEV))
    d = {n: None if t is None else put(n, t) for n, t in i.items()}
    dt, n = i["x"].dtype, i["weight"].shape[0]
    rows = i["x"].shape[0]
    factor = R.keep_factor(p, i["state"], rows, n).to(where)
    args = dict(activation=act, gate=d["gate"], dropout=p, state=d["state"])
    y, kept = ops.linear_fwd(d["x"], d["weight"], d["bias"], residual=d["residual"], out_dtype=out_dtype, keep=True, **args)
    x, w, b, g, res, dy = double(where, *(i[k] for k in ("x", "weight", "bias", "gate", "residual", "dy")))
    ref = R.linear(x, w, b, act, g, res, factor)
    assert kept.dtype == dt and y.dtype == (i["residual"].dtype if res is not None else out_dtype or dt)
    close(kept, ref["kept"][0], R.rounded(*ref["kept"], dt), "kept")
    close(y, ref["y"][0], R.rounded(*ref["y"], y.dtype), "y")
    assert torch.equal(y, ops.linear_fwd(d["x"], d["weight"], d["bias"], residual=d["residual"], out_dtype=out_dtype,
                                         **args))
    grads = ops.linear_bwd(d["dy"], d["x"], d["weight"], kept, **args)
    ref = R.linear_bwd(dy, x, w, kept.double().to(where), act, g, factor, dt)
    pdt = dt if i["gate"] is None else i["gate"].dtype
    for name, got, kind in zip(("dx", "dweight", "dbias", "dgate"), grads, (dt, dt, pdt, pdt)):
        if name == "dgate" and g is None:
            assert got is None
            continue
        assert got.dtype == kind
        close(got, ref[name][0], R.rounded(*ref[name], kind), name)
    again = ops.linear_bwd(d["dy"], d["x"], d["weight"], kept, **args)
    assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(grads, again))


SIZES = [(1, 8, 8), (1, 64, 16), (2, 72, 24), (5, 1024, 128), (16, 200, 40), (17, 512, 130), (32, 4096, 64), (33, 96, 264),
         (64, 128, 1000), (65, 128, 8), (127, 64, 128), (128, 136, 128), (129, 1024, 136), (261, 1024, 256), (300, 56, 515),
         (520, 264, 1024)]


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_linear(ops, dt, rows, k, n):
    check(ops, inputs(rows, k, n, dt, gate=False))


@pytest.mark.parametrize("rows,k,n", SIZES[::2])
@pytest.mark.parametrize("act,p,residual", [("gelu", 0.0, None), ("gelu_tanh", 0.1, BF), (None, 0.5, F32), ("gelu", 0.3, F32)])
def test_epilogue(ops, rows, k, n, act, p, residual):
    check(ops, inputs(rows, k, n, BF, seed=1, residual=residual), act, p)


@pytest.mark.parametrize("rows,k,n", [(3, 7, 5), (1, 1, 1), (70, 65, 63), (40, 1027, 515), (200, 130, 257), (150, 9, 1030)])
@pytest.mark.parametrize("dt", [BF, FP])
def test_widths_that_8_does_not_divide(ops, rows, k, n, dt):
    check(ops, inputs(rows, k, n, dt, seed=2, residual=dt), "gelu")
    check(ops, inputs(rows, k, n, dt, seed=3, gate=False), None)


@pytest.mark.parametrize("pdt", [F32, BF, FP])
@pytest.mark.parametrize("dt", [BF, FP])
def test_parameter_types(ops, dt, pdt):
    check(ops, inputs(50, 64, 72, dt, seed=4, pdt=pdt, residual=F32), "gelu", 0.2)
    check(ops, inputs(200, 64, 72, dt, seed=5, pdt=pdt), None)
    check(ops, inputs(20, 64, 72, dt, seed=6, pdt=pdt, bias=False, gate=False), None)


def test_fp32_result(ops):
    check(ops, inputs(40, 128, 48, BF, seed=7, ydt=F32), "gelu", 0.0, F32)
    check(ops, inputs(140, 128, 48, BF, seed=7, ydt=F32, gate=False), None, 0.0, F32)


@pytest.mark.parametrize("rows,k,n", [(3100, 72, 4096), (6401, 8, 2000)])
def test_tiles_of_256_rows(ops, rows, k, n):
    """Enough tiles for the larger ones without a split."""
    check(ops, inputs(rows, k, n, BF, seed=8), "gelu", 0.1)


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("rows,k,n", [(4001, 1030, 2050), (10411, 1544, 6150), (10901, 4104, 1000), (70003, 72, 130),
                                      (5000, 520, 1030)])
def test_ragged_tiles_of_every_size(ops, rows, k, n, dt):
    """Tiles of 64 to 256 rows and columns that end inside the matrices, in all three products, with reductions that 64 does
    not divide (the formulas in 64 bits on the GPU)."""
    check(ops, inputs(rows, k, n, dt, seed=30, gate=False), None, where=DEV)
    check(ops, inputs(rows, k, n, dt, seed=31, residual=F32), "gelu", 0.1, where=DEV)


@pytest.mark.parametrize("rows", [1, 2, 3])
@pytest.mark.parametrize("k,n", [(64, 64), (128, 4096), (192, 72), (256, 1000), (320, 128)])
def test_few_steps(ops, rows, k, n):
    """Reductions of one to five steps over few to many rows."""
    check(ops, inputs(64 * rows + 1, k, n, BF, seed=32), "gelu")


@pytest.mark.parametrize("rows,k,n", [(130, 4104, 136), (70, 2048, 64)])
def test_split_reductions(ops, rows, k, n):
    check(ops, inputs(rows, k, n, BF, seed=9, residual=F32), "gelu_tanh", 0.1)


def test_long_reduction_over_rows(ops):
    """The weight's gradient sums over many rows, split among work-groups."""
    check(ops, inputs(20011, 40, 24, BF, seed=10, gate=False))
    check(ops, inputs(9001, 130, 70, FP, seed=11), "gelu")


def test_offsets_beyond_32_bits(ops):
    """Operands and results of more than 2^31 elements: rows from both ends against 64 bits, the sums over all rows."""
    rows, wide, narrow = 530_011, 4104, 72
    g = torch.Generator(device=DEV).manual_seed(6)

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=BF)
    far = torch.cat([torch.arange(3), torch.arange(rows - 130, rows)]).to(DEV)
    state = torch.tensor([9, 1], device=DEV)
    keep = torch.cat([R.keep_bits((9, 1), 3, wide), R.keep_bits((9, 1), 130, wide, rows - 130)]).to(DEV)
    for k, n in ((wide, narrow), (narrow, wide)):
        x, w = rnd(rows, k), rnd(n, k) / math.sqrt(k)
        y = ops.linear_fwd(x, w, dropout=0.25 if n == wide else 0.0, state=state)
        factor = (keep >= 16384).double() * (4 / 3) if n == wide else 1.0
        z, z_tol = R.linear(x[far].double(), w.double(), None, None, None, None, torch.ones(1, 1, device=DEV))["kept"]
        close(y[far], z * factor, R.rounded(z * factor, (z_tol + 4 * R.E32 * z.abs()) * factor, BF), "y")
        dy = rnd(rows, n)
        dx, dw, db, _ = ops.linear_bwd(dy, x, w)
        d = dy[far].double()
        want, tol = d @ w.double(), (n + 2) * R.E32 * (d.abs() @ w.double().abs())
        close(dx[far], want, R.rounded(want, tol, BF), "dx")
        want = torch.zeros(n, k, dtype=torch.float64, device=DEV)
        size = torch.zeros_like(want)
        for a, b in zip(dy.split(65536), x.split(65536)):
            want += a.double().t().contiguous() @ b.double()
            size += a.double().abs().t().contiguous() @ b.double().abs()
        # (sums of half a million products: the bound of n * 2^-24 is a tenth of them; these are split, of random sign, and
        # held to 2^-10 of their magnitudes, a sixtieth of that bound)
        close(dw, want, R.rounded(want, 2.0 ** -10 * size, BF), "dweight")
        del x, w, y, dy, dx


@pytest.mark.parametrize("p", [0.0, 0.5, 1.0])
def test_all_kept_and_all_dropped(ops, p):
    check(ops, inputs(70, 64, 72, BF, seed=12, residual=F32), "gelu", p)


def test_layouts(ops):
    """Views with strides, offsets that break the alignment, batches of rows."""
    i = inputs(48, 96, 104, BF, seed=13, residual=F32)

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
    for put in (wide, odd, turned):
        check(ops, i, "gelu", 0.1, put=put)
    x, w = i["x"].to(DEV), i["weight"].to(DEV)
    y = ops.linear_fwd(x, w)
    assert torch.equal(ops.linear_fwd(x.view(4, 3, 4, 96), w), y.view(4, 3, 4, 104))
    assert torch.equal(ops.linear_fwd(x[7], w), ops.linear_fwd(x[7:8], w)[0])


def test_broadcast_gradient(ops):
    i = inputs(33, 64, 72, BF, seed=14)
    x, w = i["x"].to(DEV), i["weight"].to(DEV)
    one = torch.ones((), dtype=BF, device=DEV).expand(33, 72)
    row = torch.randn(72, device=DEV).to(BF).expand(33, 72)
    for dy in (one, row):
        for a, b in zip(ops.linear_bwd(dy, x, w)[:3], ops.linear_bwd(dy.contiguous(), x, w)[:3]):
            assert torch.equal(a, b)


def test_no_rows(ops):
    x, w = torch.zeros(0, 24, dtype=BF, device=DEV), torch.ones(16, 24, dtype=BF, device=DEV)
    y, kept = ops.linear_fwd(x, w, keep=True)
    assert y.shape == kept.shape == (0, 16)
    dx, dw, db, _ = ops.linear_bwd(y, x, w)
    assert dx.shape == (0, 24) and dw.shape == (16, 24) and (dw == 0).all() and (db == 0).all()
    dw = ops.linear_bwd(y, x, w, need=(False, True, False, False), weight_dtype=F32)[1]
    assert dw.dtype == F32 and (dw == 0).all()


def test_only_what_is_needed(ops):
    i = inputs(70, 64, 72, BF, seed=15)
    d = {n: None if t is None else t.to(DEV) for n, t in i.items()}
    _, kept = ops.linear_fwd(d["x"], d["weight"], d["bias"], "gelu", d["gate"], keep=True)
    every = ops.linear_bwd(d["dy"], d["x"], d["weight"], kept, "gelu", d["gate"])
    for which in range(16):
        need = tuple(bool(which >> j & 1) for j in range(4))
        some = ops.linear_bwd(d["dy"], d["x"], d["weight"], kept, "gelu", d["gate"], need=need)
        for n, a, b in zip(need, some, every):
            assert (a is not None) == n and (not n or torch.equal(a, b))
    wide = ops.linear_bwd(d["dy"], d["x"], d["weight"], kept, "gelu", d["gate"], weight_dtype=F32)[1]
    assert wide.dtype == F32 and torch.equal(wide.to(BF), every[1])


def test_values_at_the_ends(ops):
    """Infinities and NaN stay in their rows; activations reach their limits."""
    x = torch.randn(40, 64).to(BF)
    w = torch.zeros(8, 64).to(BF)
    w[0, 0], w[1, 0], w[2, 1] = 1, -1, 1
    x[:, 0] = 0
    x[3, 0], x[4, 0], x[5, 1] = 300.0, math.inf, math.nan
    for act in ("gelu", "gelu_tanh"):
        y, kept = ops.linear_fwd(x.to(DEV), w.to(DEV), activation=act, keep=True)
        y, kept = y.cpu().float(), kept.cpu().float()
        assert y[3, 0] == 300 and y[3, 1] == 0
        assert kept[5].isnan().all() and y[5].isnan().all()  # (a NaN times a zero weight too)
        assert y[4, 0] == math.inf and y[4, 1] == 0 and y[4, 2:].isnan().all()
        rest = torch.ones(40, dtype=torch.bool)
        rest[4:6] = False
        assert y[rest].isfinite().all()
        slope = ops.linear_bwd(torch.ones(40, 8).to(BF).to(DEV), x.to(DEV), w.to(DEV), kept.to(BF).to(DEV), act,
                               need=(True, False, False, False))[0].cpu().float()
        assert slope[3, 0] == 1.0 and slope[5].isnan().any() and slope[rest].isfinite().all()


@pytest.mark.parametrize("act", [None, "gelu", "gelu_tanh"])
@pytest.mark.parametrize("rows,k,n", [(20, 64, 72), (300, 40, 130)])
def test_infinities_in_dropped_places(ops, act, rows, k, n):
    """What a dropped element holds reaches neither the result nor a gradient."""
    i = inputs(rows, k, n, BF, 9)
    dropped = R.keep_factor(0.5, i["state"], rows, n) == 0
    x = i["x"].clone()
    x[3] = math.inf  # (row 3 is infinities or NaN before the mask)
    y = ops.linear_fwd(x.to(DEV), i["weight"].to(DEV), None, act, None, i["residual"], None, 0.5, i["state"].to(DEV)).cpu()
    assert (y[3][dropped[3]] == 0).all() and not y[3][~dropped[3]].isfinite().all()
    kept = torch.randn(rows, n, generator=torch.Generator().manual_seed(1)).to(BF)
    res = []
    for value in (1.0, math.inf, -math.inf, math.nan):
        z = torch.where(dropped, torch.tensor(value, dtype=BF), kept)
        res.append(ops.linear_bwd(i["dy"].to(DEV), i["x"].to(DEV), i["weight"].to(DEV), z.to(DEV), act, i["gate"].to(DEV), 0.5,
                                  i["state"].to(DEV)))
    for other in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(res[0], other))


def test_gradients_by_differences(ops):
    """The gradient of <y, dy> along random directions against differences of the forward kernel in fp32 results; the inputs
    are multiples of 2^-6, so that moved inputs are exact."""
    g = torch.Generator().manual_seed(5)

    def grid(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale * 64).round().clamp(-127, 127).div(64)
    x, w, b, gate = grid(70, 48), grid(56, 48, scale=0.15), grid(56, scale=0.3), grid(56, scale=0.5)
    dy = grid(70, 56)
    state = torch.tensor([3, 4], device=DEV)

    def f(x, w, b, gate):
        y = ops.linear_fwd(x.to(BF).to(DEV), w.to(BF).to(DEV), b.to(DEV), "gelu", gate.to(DEV), out_dtype=F32, dropout=0.25,
                           state=state)
        return float((y.double() * dy.to(DEV).double()).sum())
    _, kept = ops.linear_fwd(x.to(BF).to(DEV), w.to(BF).to(DEV), b.to(DEV), "gelu", gate.to(DEV), dropout=0.25, state=state,
                             keep=True)
    grads = ops.linear_bwd(dy.to(DEV), x.to(BF).to(DEV), w.to(BF).to(DEV), kept, "gelu", gate.to(DEV), 0.25, state,
                           weight_dtype=F32)
    args = [x, w, b, gate]
    for which, grad in enumerate(grads):
        step = torch.sign(torch.randn(args[which].shape, generator=g)) * 2.0 ** -6
        up, down = list(args), list(args)
        up[which], down[which] = args[which] + step, args[which] - step
        slope = float((grad.double().cpu() * step.double()).sum())
        diff = (f(*up) - f(*down)) / 2
        # kept and dz carry bf16 roundings (2^-9 each, of random sign), the difference a third derivative of step^2 / 6 of
        # sums whose z moves by up to 48 * 2^-6 * 0.4: a few per cent of the magnitudes that are summed
        size = float((grad.double().cpu() * step.double()).abs().pow(2).sum().sqrt())
        assert abs(slope - diff) <= 0.15 * size + 0.02 * abs(diff), (which, slope, diff, size)


def test_streams_and_graph(ops):
    """On a side stream, and captured and replayed with eager work between the replays."""
    i = inputs(300, 512, 136, BF, seed=16, residual=F32)
    d = {n: None if t is None else t.to(DEV) for n, t in i.items()}

    def step():
        args = dict(activation="gelu", gate=d["gate"], dropout=0.1, state=d["state"])
        y, kept = ops.linear_fwd(d["x"], d["weight"], d["bias"], residual=d["residual"], keep=True, **args)
        return (y, kept, *ops.linear_bwd(d["dy"], d["x"], d["weight"], kept, **args))
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
        d["x"].copy_(inputs(300, 512, 136, BF, seed=20 + seed)["x"])
        d["state"].add_(1)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        assert not torch.equal(got[0], want[0])
