"""LayerNorm and the rotary head norm with their gradients (``ops.layer_norm_fwd`` / ``_bwd``, ``ops.head_rotary_fwd`` /
``_bwd``) against the formulas in 64 bits."""
import importlib
import math

import pytest
import torch

import train_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF, FP = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return importlib.import_module(pkg.__name__ + ".ops")


def close(got, want, tol, name):
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} off, worst {float((err / tol)[bad].max()):.3g} x the bound"


def norm_bounds(x, dy, w, b, eps, D):
    """fp64 LayerNorm, its gradients per row, and bounds without the result's rounding. Errors of the statistics: sums of
    D terms (D * 2^-24 of their magnitudes, one more rounding each step)."""
    y, m, r, xh = R.layer_norm(x, w, b, eps)
    e = R.E32
    m_tol = (D + 2) * e * x.abs().mean(-1, keepdim=True)
    c = x - m[..., None]
    # a centred value: the mean's error and its own rounding; the variance: twice that, D more roundings
    c_tol = m_tol + e * (c.abs() + x.abs())
    var = (c * c).mean(-1, keepdim=True)
    v_tol = 2 * (c.abs() * c_tol).mean(-1, keepdim=True) + (D + 4) * e * var + e * eps
    r_rel = 0.5 * v_tol / (var + eps) + 4 * e  # first order; the cases keep it far below 1
    xh_tol = r[..., None] * c_tol + xh.abs() * (r_rel + 2 * e)
    wa = 1.0 if w is None else w.abs()
    y_tol = xh_tol * wa + 4 * e * (xh.abs() * wa + (0 if b is None else b.abs()))
    res = {"y": (y, y_tol), "mean": (m, m_tol[..., 0]), "rstd": (r, (r[..., None] * r_rel)[..., 0] + e * r)}
    if dy is None:
        return res
    g = dy if w is None else dy * w
    dx = R.layer_norm_bwd(dy, xh, r, w)
    ga = g.abs()
    m1_tol = (D + 3) * e * ga.mean(-1, keepdim=True)
    m2_tol = (D + 4) * e * (ga * xh.abs()).mean(-1, keepdim=True) + (ga * xh_tol).mean(-1, keepdim=True)
    m2 = (g * xh).mean(-1, keepdim=True)
    inner = e * 4 * (ga + g.mean(-1, keepdim=True).abs() + (xh * m2).abs())
    dx_tol = r[..., None] * (inner + m1_tol + xh.abs() * m2_tol + xh_tol * m2.abs()) + dx.abs() * (r_rel + 4 * e)
    dw, dw_tol = dy * xh, dy.abs() * xh_tol  # to be summed over rows
    res.update(dx=(dx, dx_tol), dw=(dw, dw_tol + 2 * e * dw.abs()), db=(dy, torch.zeros_like(dy)))
    return res


def rounded(value, tol, dtype):
    """The bound after the one rounding to dtype (fp16: also half of its smallest step)."""
    return tol * (1 + 2 * R.half_step(dtype)) + R.half_step(dtype) * value.abs() + (2.0 ** -25 if dtype == FP else 1e-37)


def summed(value, tol, dims, dtype):
    n = math.prod(value.shape[d] for d in dims)
    s = value.sum(dims)
    return s, rounded(s, tol.sum(dims) + (n + 2) * R.E32 * value.abs().sum(dims), dtype)


# ---- LayerNorm ------------------------------------------------------------------------------------------

def norm_inputs(shape, dt, out, seed, affine=True, pdt=F32):
    g = torch.Generator().manual_seed(seed)
    D = shape[-1]
    x = torch.randn(shape, generator=g) * (0.5 + 2 * torch.rand(*shape[:-1], 1, generator=g)) + 0.7
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(pdt) if affine else None
    b = (0.2 * torch.randn(D, generator=g)).to(pdt) if affine else None
    return x.to(dt), torch.randn(shape, generator=g).to(out), w, b


def gpu(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def check_norm(ops, x, dy, w, b, out_dtype, eps=1e-5):
    gx, gdy, gw, gb = gpu(x, dy, w, b)
    y, mean, rstd = ops.layer_norm_fwd(gx, gw, gb, eps=eps, out_dtype=out_dtype)
    dx, dw, db = ops.layer_norm_bwd(gdy, gx, mean, rstd, gw)
    D = x.shape[-1]
    ref = norm_bounds(x.double(), dy.double(), None if w is None else w.double(), None if b is None else b.double(),
                      eps, D)
    assert y.dtype == (out_dtype or x.dtype) and dx.dtype == x.dtype
    close(mean, ref["mean"][0], ref["mean"][1] + 1e-37, "mean")
    close(rstd, *ref["rstd"], "rstd")
    close(y, ref["y"][0], rounded(*ref["y"], y.dtype), "y")
    close(dx, ref["dx"][0], rounded(*ref["dx"], dx.dtype), "dx")
    dims = tuple(range(x.dim() - 1))
    pd = F32 if w is None else w.dtype
    assert dw.dtype == db.dtype == pd
    close(dw, *summed(*ref["dw"], dims, pd), "dw")
    close(db, *summed(*ref["db"], dims, pd), "db")
    return y, mean, rstd, dx, dw, db


@pytest.mark.parametrize("dt,out", [(BF, BF), (FP, FP), (F32, F32), (F32, BF), (F32, FP)])
@pytest.mark.parametrize("rows,dim", [(1, 8), (3, 64), (70, 128), (33, 200), (129, 512), (65, 1024), (17, 1536),
                                      (9, 2048), (11, 4096), (5, 8192), (41, 2), (130, 63), (19, 65), (7, 513),
                                      (9, 1027), (6, 2047), (5, 2049), (3, 8191)])
def test_layer_norm(ops, dt, out, rows, dim):
    x, dy, w, b = norm_inputs((rows, dim), dt, out, rows + dim)
    check_norm(ops, x, dy, w, b, out if out != dt else None)


@pytest.mark.parametrize("affine,pdt", [(False, F32), (True, BF), (True, FP)])
def test_layer_norm_parameters(ops, affine, pdt):
    x, dy, w, b = norm_inputs((2, 50, 96), BF, BF, 1, affine, pdt)
    check_norm(ops, x, dy, w, b, None)
    x, dy, w, b = norm_inputs((700, 33), F32, F32, 2, affine, pdt)
    check_norm(ops, x, dy, w, b, None)


def test_layer_norm_many_rows(ops):
    """More rows than one step of every work-group."""
    x, dy, w, b = norm_inputs((30011, 64), BF, BF, 5)
    check_norm(ops, x, dy, w, b, None)
    x, dy, w, b = norm_inputs((9001, 129), F32, BF, 6)
    check_norm(ops, x, dy, w, b, BF)


def test_layer_norm_one_value(ops):
    """Rows of one element, and constant rows: the variance is zero."""
    x = torch.full((5, 1), 3.0)
    y, mean, rstd = ops.layer_norm_fwd(x.to(DEV), eps=1e-5)
    assert (y == 0).all() and (mean == 3).all() and torch.allclose(rstd.cpu(), torch.full((5,), 1e-5) ** -0.5)
    x = torch.full((5, 128), -2.5).to(BF)
    w = torch.ones(128)
    y, mean, rstd = ops.layer_norm_fwd(x.to(DEV), w.to(DEV), w.to(DEV))
    assert (y == 1).all() and (mean == -2.5).all()


def test_layer_norm_strided_rows_and_empty(ops):
    x, dy, w, b = norm_inputs((37, 192), BF, BF, 3)
    want = check_norm(ops, x, dy, w, b, None)
    gw, gb = gpu(w, b)
    for pad in (8, 3):  # rows of a wider buffer: vectors, then single elements
        wide = torch.zeros(37, 192 + pad, dtype=BF, device=DEV)
        gx = wide[:, pad:].copy_(x)
        y, mean, rstd = ops.layer_norm_fwd(gx, gw, gb)
        gdy = torch.zeros(37, 192 + pad, dtype=BF, device=DEV)[:, :192].copy_(dy)
        dx, dw, db = ops.layer_norm_bwd(gdy, gx, mean, rstd, gw)
        for a, c in zip((y, dx), (want[0], want[3])):
            # the same formulas with another order of the sums: one step of the rounding at most
            assert (a.float() - c.float()).abs().max() <= 2 ** -7 * c.float().abs().max()
        if pad == 8:
            assert torch.equal(y, want[0]) and torch.equal(dx, want[3]) and torch.equal(dw, want[4])
    t = x.to(DEV).t().contiguous().t()  # columns first: copied
    assert torch.equal(ops.layer_norm_fwd(t, gw, gb)[0], want[0])
    e = torch.empty(0, 192, dtype=BF, device=DEV)
    y, mean, rstd = ops.layer_norm_fwd(e, gw, gb)
    dx, dw, db = ops.layer_norm_bwd(e, e, mean, rstd, gw)
    assert y.shape == dx.shape == e.shape and (dw == 0).all() and (db == 0).all()


def test_layer_norm_some_gradients(ops):
    x, dy, w, b = norm_inputs((20, 64), BF, BF, 3)
    gx, gdy, gw, gb = gpu(x, dy, w, b)
    y, mean, rstd = ops.layer_norm_fwd(gx, gw, gb)
    full = ops.layer_norm_bwd(gdy, gx, mean, rstd, gw)
    for need in ((False, False), (True, False), (False, True)):
        dx, dw, db = ops.layer_norm_bwd(gdy, gx, mean, rstd, gw, need_params=need)
        assert torch.equal(dx, full[0])
        for t, f, n in ((dw, full[1], need[0]), (db, full[2], need[1])):
            assert (t is None) == (not n) and (t is None or torch.equal(t, f))


# ---- rotary positions -----------------------------------------------------------------------------------

def rotary_inputs(B, N, G, H, D, axes, positions, R, dt, seed, pos_dt=torch.int64, norm=True, pdt=F32):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, N, G, H, D, generator=g) * 1.5 + 0.3).to(dt)
    dy = torch.randn(B, N, G, H, D, generator=g).to(dt)
    pos = torch.randint(0, positions, (B, N, axes), generator=g).to(pos_dt)
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * 50.0 ** -(torch.arange(0, R // axes, 2) / (R // axes))
    w = (1 + 0.3 * torch.randn(G, D, generator=g)).to(pdt) if norm else None
    b = (0.2 * torch.randn(G, D, generator=g)).to(pdt) if norm else None
    return x, dy, pos, ang.cos().float(), ang.sin().float(), w, b


def check_rotary(ops, x, dy, pos, cos, sin, w, b, layout, R_dim, norm, eps=1e-6, views=False):
    gx, gdy, gpos, gcos, gsin, gw, gb = gpu(x, dy, pos, cos, sin, w, b)
    if views:  # q and k of a qkv buffer, dx into another
        B, N, G, H, D = x.shape
        gx = torch.zeros(B, N, G + 1, H, D, dtype=x.dtype, device=DEV)[:, :, :G].copy_(gx)
        buf = torch.full((B, N, G + 1, H, D), 5.0, dtype=x.dtype, device=DEV)
    args = dict(pos=gpos, tables=(gcos, gsin), layout=layout, rotary_dim=R_dim) if pos is not None else {}
    y = ops.head_rotary_fwd(gx, norm=norm, weight=gw, bias=gb, eps=eps, **args)
    dx, dw, db = ops.head_rotary_bwd(gdy, gx, norm=norm, weight=gw, eps=eps, out=buf[:, :, :G] if views else None, **args)
    if views:
        assert (buf[:, :, G] == 5).all()
    X, DY = x.double(), dy.double()
    W, Bb = (None if t is None else t.double()[:, None] for t in (w, b))
    e, D = R.E32, x.shape[-1]
    dy0 = DY if pos is None else R.rotate(DY, pos, cos, sin, layout, R_dim, -1.0)
    turn = (lambda t: t) if pos is None else (lambda t: R.rotate(t, pos, cos.abs(), -sin.abs(), layout, R_dim).abs()
                                              + R.rotate(t, pos, cos.abs(), sin.abs(), layout, R_dim).abs())
    dy0_tol = 3 * e * turn(DY.abs())
    if norm:
        ref = norm_bounds(X, dy0, W, Bb, eps, D)
        y0, y0_tol = ref["y"]
        # the rotated gradient's own error passes on like a gradient, of magnitude at most that of its bound
        more = norm_bounds(X, dy0_tol, None if W is None else W.abs(), None, eps, D)
        r, xh = ref["rstd"][0][..., None], R.layer_norm(X, None, None, eps)[3].abs()
        gt = dy0_tol * (1 if W is None else W.abs())
        extra = r * (gt + gt.mean(-1, keepdim=True) + xh * (gt * xh).mean(-1, keepdim=True))
        want_dx, dx_tol = ref["dx"][0], ref["dx"][1] + extra + more["dx"][1]
    else:
        y0, y0_tol, want_dx, dx_tol = X, torch.zeros_like(X), dy0, dy0_tol
    want = y0 if pos is None else R.rotate(y0, pos, cos, sin, layout, R_dim)
    y_tol = 3 * e * turn(y0.abs()) + turn(y0_tol)
    close(y, want, rounded(want, y_tol, x.dtype), "y")
    close(dx, want_dx, rounded(want_dx, dx_tol, x.dtype), "dx")
    if norm:
        pd = F32 if w is None else w.dtype
        dims = (0, 1, 3)
        close(dw, *summed(ref["dw"][0], ref["dw"][1] + dy0_tol * xh, dims, pd), "dw")
        close(db, *summed(dy0, dy0_tol, dims, pd), "db")
    else:
        assert dw is None and db is None
    return y, dx, dw, db


@pytest.mark.parametrize("dt", [BF, FP, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,N,G,H,D,axes,R", [(1, 1, 1, 1, 64, 2, 64), (2, 37, 2, 16, 64, 2, 64), (1, 130, 2, 3, 64, 1, 32),
                                              (3, 5, 1, 24, 128, 1, 64), (1, 70, 3, 2, 96, 2, 48), (2, 9, 2, 5, 32, 2, 16),
                                              (1, 33, 2, 2, 40, 3, 36), (1, 11, 1, 3, 6, 1, 4), (2, 7, 2, 2, 126, 1, 126),
                                              (1, 300, 2, 1, 2, 1, 2)])
def test_rotary(ops, dt, layout, B, N, G, H, D, axes, R):
    for norm in (True, False):
        args = rotary_inputs(B, N, G, H, D, axes, 60, R, dt, B + N + D, norm=norm,
                             pos_dt=torch.int64 if norm else torch.int32)
        check_rotary(ops, *args, layout, R, norm, views=norm)


def test_norm_without_rotation(ops):
    x, dy, _, _, _, w, b = rotary_inputs(2, 50, 2, 4, 64, 1, 4, 64, BF, 3)
    check_rotary(ops, x, dy, None, None, None, w, b, "half", None, True)
    check_rotary(ops, x, dy, None, None, None, None, None, "half", None, True)


@pytest.mark.parametrize("pdt", [BF, FP])
def test_rotary_parameter_types(ops, pdt):
    check_rotary(ops, *rotary_inputs(1, 40, 2, 4, 64, 2, 30, 64, BF, 4, pdt=pdt), "half", 64, True)


def test_rotary_without_eps(ops):
    """No eps, and rows that fill no step: the lanes without a row add nothing to the parameters' gradients."""
    for N in (1, 2, 43):
        check_rotary(ops, *rotary_inputs(1, N, 2, 3, 64, 2, 30, 64, BF, 8 + N), "half", 64, True, eps=0.0)


def test_rotary_many_rows(ops):
    """More rows than one step of every work-group."""
    check_rotary(ops, *rotary_inputs(2, 4100, 2, 3, 32, 2, 40, 32, BF, 6), "half", 32, True)


def test_positions_outside_the_tables(ops):
    x, dy, pos, cos, sin, w, b = rotary_inputs(1, 20, 1, 2, 64, 2, 30, 64, BF, 2)
    for dt in (torch.int32, torch.int64):
        far = pos.to(dt).clone()
        far[0, :5] = -3
        far[0, 5:9] = torch.iinfo(dt).max
        far[0, 9] = 30
        check_rotary(ops, x, dy, far, cos, sin, w, b, "half", 64, True)  # (the reference clamps)


def test_odd_strides_and_layouts(ops):
    """Rows that vectors cannot read, expanded heads, tokens in another order of the dimensions."""
    x, dy, pos, cos, sin, w, b = rotary_inputs(2, 12, 2, 4, 64, 2, 30, 64, BF, 8)
    want = check_rotary(ops, x, dy, pos, cos, sin, w, b, "half", 64, True)
    gx, gdy, gpos, gcos, gsin, gw, gb = gpu(x, dy, pos, cos, sin, w, b)
    args = dict(pos=gpos, tables=(gcos, gsin), norm=True, weight=gw, eps=1e-6)
    perm = gx.permute(2, 3, 1, 0, 4).contiguous().permute(3, 2, 0, 1, 4)
    assert torch.equal(ops.head_rotary_fwd(perm, bias=gb, **args), want[0])
    odd = torch.zeros(2, 12, 2, 4, 67, dtype=BF, device=DEV)[..., 2:66].copy_(gx)
    y = ops.head_rotary_fwd(odd, bias=gb, **args)
    assert (y.float() - want[0].float()).abs().max() <= 2 ** -7 * want[0].float().abs().max()
    back = gx.flip(-1).contiguous().flip(-1)  # (a copy: torch has no negative strides)
    assert torch.equal(ops.head_rotary_fwd(back, bias=gb, **args), want[0])
    one = gx[:, :, :, :1].expand(-1, -1, -1, 4, -1)
    assert torch.equal(ops.head_rotary_fwd(one, bias=gb, **args)[:, :, :, 3], want[0][:, :, :, 0])
    last = gx.permute(4, 0, 1, 2, 3).contiguous().permute(1, 2, 3, 4, 0)
    assert torch.equal(ops.head_rotary_fwd(last, bias=gb, **args), want[0])
    assert torch.equal(ops.head_rotary_bwd(gdy, last, **args)[0], want[1])


def test_rotary_empty(ops):
    for shape in ((0, 5, 2, 3, 64), (2, 0, 2, 3, 64)):
        x = torch.empty(shape, dtype=BF, device=DEV)
        pos = torch.empty(*shape[:2], 2, dtype=torch.int64, device=DEV)
        tables = ops.rotary_tables(10, 32, device=DEV)
        w = torch.ones(2, 64, device=DEV)
        assert ops.head_rotary_fwd(x, pos, tables, norm=True, weight=w).shape == x.shape
        dx, dw, db = ops.head_rotary_bwd(x, x, pos, tables, norm=True, weight=w)
        assert dx.shape == x.shape and (dw == 0).all() and (db == 0).all()


def test_far_positions(ops):
    """Tables of 2^20 positions: angles from 64 bits, the rotation within fp32 roundings of the exact one."""
    n = 1 << 20
    cos, sin = ops.rotary_tables(n, 64, base=10000.0, device=DEV)
    j = torch.arange(0, 64, 2, dtype=torch.float64) / 64
    pos = torch.tensor([0, 1, 65535, n - 2, n - 1])
    ang = pos[:, None].double() * 10000.0 ** -j
    assert (cos.cpu()[pos].double() - ang.cos()).abs().max() <= 2.0 ** -24  # 1 rounded once, and pow's last bit
    assert (sin.cpu()[pos].double() - ang.sin()).abs().max() <= 2.0 ** -24
    x = torch.randn(1, 5, 1, 2, 64, generator=torch.Generator().manual_seed(0))
    y = ops.head_rotary_fwd(x.to(DEV), pos[None, :, None].to(DEV), (cos, sin))
    u, v = x[..., :32].double(), x[..., 32:].double()
    c, s = ang.cos()[None, :, None, None], ang.sin()[None, :, None, None]
    want = torch.cat([u * c - v * s, v * c + u * s], -1)
    tol = 5 * R.E32 * torch.cat([u.abs() + v.abs()] * 2, -1)
    close(y, want, tol + 1e-30, "y")


def test_graph_streams_and_equal_bits(ops):
    """Both operators on a side stream, captured and replayed with new inputs, and twice the same."""
    xs = rotary_inputs(2, 300, 2, 4, 64, 2, 30, 64, BF, 8)
    gx, gdy, gpos, gcos, gsin, gw, gb = gpu(*xs)
    nx, ndy, nw, nb = gpu(*norm_inputs((900, 256), F32, BF, 2))

    def run():
        a = dict(pos=gpos, tables=(gcos, gsin), norm=True, weight=gw)
        y = ops.head_rotary_fwd(gx, bias=gb, **a)
        ny, mean, rstd = ops.layer_norm_fwd(nx, nw, nb, out_dtype=BF)
        return (y, *ops.head_rotary_bwd(gdy, gx, **a), ny, *ops.layer_norm_bwd(ndy, nx, mean, rstd, nw))
    want = run()
    assert all(torch.equal(a, b) for a, b in zip(want, run()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for seed in (1, 2, 3):
        gx.copy_(rotary_inputs(2, 300, 2, 4, 64, 2, 30, 64, BF, seed)[0])
        nx.copy_(norm_inputs((900, 256), F32, BF, seed)[0])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held)), seed
