"""Attention over frames with its gradients (``ops.frame_attn_fwd`` / ``frame_attn_bwd``) against the formulas in
64 bits: patterns, frame sizes around the tiles, masks, strides, devices' streams, capture and replay."""
import importlib
import math

import pytest
import torch

import train_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return importlib.import_module(pkg.__name__ + ".ops")


def patterns_of(ops, name, H):
    kinds = {"dense": (ops.DENSE,), "local": (ops.FRAME_LOCAL,), "anchor_local": (ops.ANCHOR_LOCAL,),
             "anchor": (ops.ANCHOR,), "skip": (ops.SKIP,),
             "mix": (ops.DENSE, ops.FRAME_LOCAL, ops.ANCHOR_LOCAL, ops.ANCHOR, ops.SKIP)}[name]
    return [kinds[h % len(kinds)] for h in range(H)]


def inputs(B, N, H, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(B, N, H, 64, generator=g) for _ in range(4))
    k = 0.6 * k + 0.8 * q  # near matches, so that some rows are nearly all on one key
    return tuple(t.to(torch.bfloat16) for t in (q * spread, k, v + 0.25, do * 0.1))


def check(ops, q, k, v, do, patterns, frames, mask=None, rest=True, scale=None):
    """Runs both directions on GPU copies and compares every element with the 64-bit bound."""
    gq, gk, gv, gdo = (t.to(DEV) for t in (q, k, v, do))
    gm = None if mask is None else mask.to(DEV)
    res = ops.frame_attn_fwd(gq, gk, gv, patterns, frames=frames, token_mask=gm, rest=rest, scale=scale)
    out, lse = res[:2]
    dq, dk, dv = ops.frame_attn_bwd(gdo, gq, gk, gv, out, lse, patterns, frames=frames, token_mask=gm, scale=scale,
                                    rest=res[2] if rest else None)
    ref = R.frame_attention(q, k, v, do, patterns, frames, mask, 0.125 if scale is None else scale)
    got = {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    for name, t in got.items():
        want, tol = ref[name]
        t = t.double().cpu()
        empty = torch.isinf(want)
        assert torch.equal(torch.isinf(t), empty), name
        err = torch.where(empty, 0.0, (t - want).abs())
        bad = err > tol
        assert not bad.any(), f"{name}: {int(bad.sum())} off, worst {float((err / tol).max()):.3g} x the bound"
    return got


@pytest.mark.parametrize("pattern", ["dense", "local", "anchor_local", "anchor", "skip", "mix"])
@pytest.mark.parametrize("B,F,T,H", [(1, 1, 1, 1), (2, 3, 1, 2), (1, 2, 5, 3), (1, 1, 63, 1), (1, 1, 64, 2), (2, 1, 65, 1),
                                     (1, 3, 127, 2), (1, 2, 129, 5), (1, 5, 40, 5), (1, 2, 300, 5), (3, 1, 257, 1)])
def test_against_64_bits(ops, pattern, B, F, T, H):
    q, k, v, do = inputs(B, F * T, H, 7 * F + T)
    check(ops, q, k, v, do, patterns_of(ops, pattern, H), F)


@pytest.mark.parametrize("kind", ["holes", "short", "no_first", "none", "one"])
@pytest.mark.parametrize("F,T", [(3, 70), (2, 261), (4, 64), (1, 9)])
def test_masks(ops, kind, F, T):
    """Removed tokens hold NaN and infinities: none of it reaches any output."""
    B, H = 2, 5
    q, k, v, do = inputs(B, F * T, H, T)
    g = torch.Generator().manual_seed(F)
    if kind == "holes":
        mask = torch.rand(B, F * T, generator=g) < 0.6
    elif kind == "short":
        mask = (torch.arange(F * T) < F * T - T // 2).expand(B, -1).clone()
        mask[1, : T // 3] = False
    elif kind == "no_first":
        mask = (torch.arange(F * T) >= T).expand(B, -1).clone()
        mask[1] = True
    elif kind == "none":
        mask = torch.zeros(B, F * T, dtype=torch.bool)
        mask[1] = True
    else:
        mask = torch.zeros(B, F * T, dtype=torch.bool)
        mask[0, F * T // 2] = mask[1, -1] = True
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(torch.bfloat16).min]).to(torch.bfloat16)
    for i, t in enumerate((q, k, v, do)):
        t[~mask] = bad[torch.randint(0, 4, t[~mask].shape, generator=g)]
    got = check(ops, q, k, v, do, patterns_of(ops, "mix", H), F, mask)
    for n in ("out", "dq", "dk", "dv"):
        assert (got[n].cpu()[~mask] == 0).all(), n


def test_views_of_a_qkv_buffer(ops):
    """q, k, v as the projection left them, grads into views of one buffer; nothing beside them is written."""
    B, F, T, H = 2, 2, 75, 3
    N = F * T
    q, k, v, do = inputs(B, N, H, 3)
    pat = patterns_of(ops, "mix", H)
    want = check(ops, q, k, v, do, pat, F)
    qkv = torch.stack([q, k, v], dim=2).to(DEV)  # [B, N, 3, H, 64]
    views = [qkv[:, :, i] for i in range(3)]
    out, lse, rest = ops.frame_attn_fwd(*views, pat, frames=F, rest=True)
    buf = torch.full((B, N + 2, 3, H + 1, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    grads = tuple(buf[:, 1:-1, i, :H] for i in range(3))
    gdo = torch.zeros(B, H, N, 64, dtype=torch.bfloat16, device=DEV).copy_(do.transpose(1, 2)).transpose(1, 2)
    ops.frame_attn_bwd(gdo, *views, out, lse, pat, frames=F, rest=rest, grads=grads)
    for n, t in zip(("dq", "dk", "dv"), grads):
        assert torch.equal(t, want[n]), n
    assert (buf[:, 0] == 7).all() and (buf[:, -1] == 7).all() and (buf[:, :, :, H] == 7).all()
    assert torch.equal(out, want["out"]) and torch.equal(lse, want["lse"])


@pytest.mark.parametrize("how", ["odd_rows", "offset", "last_dim", "expanded"])
def test_other_strides(ops, how):
    """Rows that no 16-byte load can read are copied; a broadcast k is read in place."""
    B, N, H = 2, 130, 2
    q, k, v, do = inputs(B, N, H, 5)
    pat = patterns_of(ops, "mix", H)
    if how == "expanded":
        k = k[:1].expand(B, -1, -1, -1)
    want = check(ops, q, k, v, do, pat, 2)
    gq, gk, gv, gdo = (t.to(DEV) for t in (q, k, v, do))
    if how == "odd_rows":
        gq = torch.zeros(B, N, H, 67, dtype=torch.bfloat16, device=DEV)[..., :64].copy_(gq)
    elif how == "offset":
        gq = torch.zeros(B * N * H * 64 + 3, dtype=torch.bfloat16, device=DEV)[3:].view(B, N, H, 64).copy_(gq)
    elif how == "last_dim":
        gq = gq.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)
    else:
        gk = gk[:1].expand(B, -1, -1, -1)
    out, lse, rest = ops.frame_attn_fwd(gq, gk, gv, pat, frames=2, rest=True)
    grads = ops.frame_attn_bwd(gdo, gq, gk, gv, out, lse, pat, frames=2, rest=rest)
    assert torch.equal(out, want["out"]) and torch.equal(lse, want["lse"])
    for n, t in zip(("dq", "dk", "dv"), grads):
        assert torch.equal(t, want[n]), n


@pytest.mark.parametrize("spread,scale", [(8.0, None), (1.0, 2.0), (0.01, 1e-3), (40.0, None)])
def test_scores_of_all_magnitudes(ops, spread, scale):
    """Scores that pass the reference of a row's first keys by far, and ones that hardly differ."""
    B, F, T, H = 1, 2, 200, 5
    q, k, v, do = inputs(B, F * T, H, 11, spread)
    if spread == 40.0:  # the scores grow along the row: the reference moves several times
        k = (k.float() * torch.linspace(0.1, 3, F * T)[None, :, None, None]).to(torch.bfloat16)
    check(ops, q, k, v, do, patterns_of(ops, "mix", H), F, scale=scale)


def test_without_rest(ops):
    """Without the rounding's rest, dq and dk carry the rounding of out (dO . out off by U of the magnitudes)."""
    B, N, H = 1, 150, 4
    q, k, v, do = inputs(B, N, H, 2)
    pat = patterns_of(ops, "dense", H)
    gq, gk, gv, gdo = (t.to(DEV) for t in (q, k, v, do))
    out, lse = ops.frame_attn_fwd(gq, gk, gv, pat)
    dq, dk, dv = ops.frame_attn_bwd(gdo, gq, gk, gv, out, lse, pat)
    ref = R.frame_attention(q, k, v, do, pat, 1)
    for b in range(B):
        for h in range(H):
            Q, K, G, o = (t[b, :, h].double() for t in (q, k, do, ref["out"][0]))
            p = torch.softmax(Q @ K.T * 0.125, -1)
            more = R.U * (G.abs() * o.abs()).sum(-1, keepdim=True) * p
            for name, t, extra in (("dq", dq, more @ K.abs() * 0.125), ("dk", dk, more.T @ Q.abs() * 0.125),
                                   ("dv", dv, torch.zeros(N, 64, dtype=torch.float64))):
                want, tol = ref[name]
                err = (t[b, :, h].double().cpu() - want[b, :, h]).abs()
                assert (err <= tol[b, :, h] + 1.01 * extra).all(), name


def test_gradients_against_differences(ops):
    """The kernels' gradients along random directions against central differences of the 64-bit loss."""
    B, F, T, H = 1, 2, 33, 5
    N = F * T
    q, k, v, do = inputs(B, N, H, 9)
    pat = patterns_of(ops, "mix", H)
    gq, gk, gv, gdo = (t.to(DEV) for t in (q, k, v, do))
    out, lse, rest = ops.frame_attn_fwd(gq, gk, gv, pat, frames=F, rest=True)
    grads = ops.frame_attn_bwd(gdo, gq, gk, gv, out, lse, pat, frames=F, rest=rest)
    base = [t.double() for t in (q, k, v)]
    tols = R.frame_attention(q, k, v, do, pat, F)
    g = torch.Generator().manual_seed(1)
    step = 1e-4
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn(B, N, H, 64, generator=g, dtype=torch.float64)
        loss = []
        for sign in (1, -1):
            x = [t + sign * step * d if j == i else t for j, t in enumerate(base)]
            loss.append((R.frame_attention(*x, do, pat, F)["out"][0] * do.double()).sum())
        want = float(loss[0] - loss[1]) / (2 * step)
        got = float((grads[i].double().cpu() * d).sum())
        # the elements' bounds along d, and the difference's own third-order term (scores move by < 0.1 step)
        assert abs(got - want) <= float((tols[name][1] * d.abs()).sum()) + 1e-4 * abs(want) + 1e-6, name


def test_runs_are_equal_bits(ops):
    q, k, v, do = (t.to(DEV) for t in inputs(2, 3 * 211, 5, 4))
    pat = patterns_of(ops, "mix", 5)

    def run():
        out, lse, rest = ops.frame_attn_fwd(q, k, v, pat, frames=3, rest=True)
        return (out, lse, rest, *ops.frame_attn_bwd(do, q, k, v, out, lse, pat, frames=3, rest=rest))
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), first))


def test_side_streams_and_two_calls_at_once(ops):
    """Calls on two streams at the same time, each with a workspace of its own."""
    pat = patterns_of(ops, "mix", 5)
    data = [tuple(t.to(DEV) for t in inputs(1, 4 * 300, 5, s)) for s in (1, 2)]

    def run(q, k, v, do):
        out, lse, rest = ops.frame_attn_fwd(q, k, v, pat, frames=4, rest=True)
        return (out, lse, *ops.frame_attn_bwd(do, q, k, v, out, lse, pat, frames=4, rest=rest))
    want = [run(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    got = []
    for _ in range(3):
        got = []
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(run(*d))
        torch.cuda.synchronize()
    for w, x in zip(want, got):
        assert all(torch.equal(a, b) for a, b in zip(w, x))


def test_captured_and_replayed(ops):
    """Both directions in a graph, replayed with new inputs between eager calls; two graphs at a time."""
    pat = patterns_of(ops, "mix", 5)

    def run(q, k, v, do):
        out, lse, rest = ops.frame_attn_fwd(q, k, v, pat, frames=2, rest=True)
        return (out, lse, *ops.frame_attn_bwd(do, q, k, v, out, lse, pat, frames=2, rest=rest))
    bufs, graphs, outs = [], [], []
    for s in (1, 2):
        b = tuple(t.to(DEV) for t in inputs(1, 2 * 150, 5, s))
        run(*b)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = run(*b)
        bufs.append(b)
        graphs.append(graph)
        outs.append(o)
    for seed in (5, 6, 7):
        for i in range(2):
            for dst, src in zip(bufs[i], inputs(1, 2 * 150, 5, seed + 10 * i)):
                dst.copy_(src)
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            want = run(*bufs[i])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, outs[i])), (seed, i)


def test_offsets_beyond_32_bits(ops):
    """Rows of a buffer whose element offsets pass 2^31 (k and v at its far end)."""
    N, H = 70, 1
    q, k, v, do = inputs(1, N, H, 8)
    pat = [ops.DENSE]
    want = check(ops, q, k, v, do, pat, 1)
    stride = (1 << 31) // 64 // 8 * 8  # elements between tokens: 70 of them pass 2^31 elements
    buf = torch.empty(N * stride, dtype=torch.bfloat16, device=DEV)
    far = [torch.as_strided(buf, (1, N, H, 64), (0, stride, 0, 1), 64 * i) for i in range(3)]
    for dst, src in zip(far, (q, k, v)):
        dst.copy_(src)
    out, lse, rest = ops.frame_attn_fwd(*far, pat, rest=True)
    dfar = [torch.as_strided(buf, (1, N, H, 64), (0, stride, 0, 1), 64 * (3 + i)) for i in range(3)]
    ops.frame_attn_bwd(do.to(DEV), *far, out, lse, pat, rest=rest, grads=dfar)
    assert torch.equal(out, want["out"])
    for n, t in zip(("dq", "dk", "dv"), dfar):
        assert torch.equal(t.contiguous(), want[n]), n


def test_no_clips(ops):
    e = torch.empty(0, 10, 2, 64, dtype=torch.bfloat16, device=DEV)
    out, lse, rest = ops.frame_attn_fwd(e, e, e, [ops.DENSE] * 2, rest=True)
    grads = ops.frame_attn_bwd(e, e, e, e, out, lse, [ops.DENSE] * 2, rest=rest)
    assert out.shape == e.shape and lse.shape == (0, 2, 10) and all(t.shape == e.shape for t in grads)


def test_long_walk_sample(ops):
    """A dense head over many tiles: sampled rows against 64 bits."""
    N, H = 12000, 2
    q, k, v, do = inputs(1, N, H, 13)
    gq, gk, gv, gdo = (t.to(DEV) for t in (q, k, v, do))
    pat = [ops.DENSE, ops.DENSE]
    out, lse, rest = ops.frame_attn_fwd(gq, gk, gv, pat, rest=True)
    dq, dk, dv = ops.frame_attn_bwd(gdo, gq, gk, gv, out, lse, pat, rest=rest)
    Q, K, V, G = (t[0, :, 1].double() for t in (gq, gk, gv, gdo))
    s = Q @ K.t().contiguous() * 0.125
    L = torch.logsumexp(s, -1)
    p = torch.exp(s - L[:, None])
    o = p @ V
    ds = p * (G @ V.t().contiguous() - (G * o).sum(-1, keepdim=True)) * 0.125
    want = {"out": o, "dq": ds @ K, "dk": ds.t().contiguous() @ Q, "dv": p.t().contiguous() @ G}
    assert (lse[0, 1].double() - L).abs().max() < 1e-5 * L.abs().max()
    for name, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        w = want[name]
        rel = float((t[0, :, 1].double() - w).norm() / w.norm())
        # a result's rounding and its operands' (P, dS, D), each at most U of magnitudes that add in quadrature
        assert rel < 2 * R.U, (name, rel)


@pytest.mark.parametrize("pattern,B,F,T,H", [("dense", 30, 1, 520, 12), ("mix", 26, 3, 190, 15), ("anchor_local", 120, 2, 65, 16),
                                             ("dense", 3, 1, 4999, 16), ("dense", 1, 1, 2060, 16), ("mix", 3, 2, 500, 12), ("mix", 1, 5, 450, 17),
                                             ("anchor_local", 2, 4, 260, 16), ("dense", 20, 1, 250, 32)])
def test_launches_of_many_rows(ops, pattern, B, F, T, H):
    """Launches of many work-groups, some of which take 64 key rows a wave: the first and the last clip against 64
    bits."""
    N = F * T
    q, k, v, do = inputs(B, N, H, T)
    pat = patterns_of(ops, pattern, H)
    gq, gk, gv, gdo = (t.to(DEV) for t in (q, k, v, do))
    out, lse, rest = ops.frame_attn_fwd(gq, gk, gv, pat, frames=F, rest=True)
    dq, dk, dv = ops.frame_attn_bwd(gdo, gq, gk, gv, out, lse, pat, frames=F, rest=rest)
    heads = range(H) if N < 1000 else range(5) if pattern == "mix" else (0, H - 1)
    for b in (0, B - 1):
        for h in heads:
            sl = (slice(b, b + 1), slice(None), slice(h, h + 1))
            ref = R.frame_attention(*(t[sl] for t in (q, k, v, do)), [pat[h]], F)
            for name, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
                want, tol = ref[name]
                err = (t[sl].double().cpu() - want).abs()
                assert (err <= tol).all(), (name, b, h, float((err / tol).max()))
            want, tol = ref["lse"]
            assert ((lse[b:b + 1, h:h + 1].double().cpu() - want).abs() <= tol)[torch.isfinite(want)].all()


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("pattern,B,F,T,H", [
    # eight waves share 32 rows and walk alone
    ("dense", 1, 1, 769, 1), ("mix", 1, 2, 500, 5), ("anchor_local", 1, 3, 600, 2), ("dense", 2, 1, 1031, 3),
    # two groups of four waves share 128 rows
    ("dense", 1, 1, 1050, 15), ("mix", 2, 3, 450, 10), ("anchor_local", 3, 2, 270, 11), ("dense", 8, 1, 513, 4)])
def test_shared_walks(ops, pattern, B, F, T, H, masked):
    """Launches of few rows and long walks, which waves or groups of waves share: odd numbers of tiles, second ranges, tiles
    that a mask empties, and a group that finds nothing."""
    N = F * T
    q, k, v, do = inputs(B, N, H, T + H, 3.0)
    mask = None
    if masked:
        g = torch.Generator().manual_seed(T)
        mask = torch.rand(B, N, generator=g) < 0.7
        mask[0, 64:256] = False
        mask[-1, N // 2:] = False
        if B > 1:
            mask[1] = False
            mask[1, 70] = True  # (one key: every other share of the walk is empty)
        for i, t in enumerate((q, k, v, do)):
            t[~mask] = (math.nan, math.inf, -math.inf, math.nan)[i]
    got = check(ops, q, k, v, do, patterns_of(ops, pattern, H), F, mask)
    if masked:
        for n in ("out", "dq", "dk", "dv"):
            assert (got[n].cpu()[~mask] == 0).all(), n


@pytest.mark.parametrize("N,H", [(5000, 1), (11000, 1), (9001, 3), (8400, 16)])
def test_long_masked_walks(ops, N, H):
    """Walks of more tiles than are looked at at once, with stretches of padding longer than that: sampled heads against
    64 bits on the GPU, in every way that a launch shares its walks."""
    q, k, v, do = (t.to(DEV) for t in inputs(1, N, H, N))
    mask = torch.rand(1, N, generator=torch.Generator().manual_seed(N)) < 0.8
    mask[0, 40: N // 2 + 77] = False
    mask[0, N - 333:] = False
    mask = mask.to(DEV)
    for t, bad in zip((q, k, v, do), (math.nan, math.inf, -math.inf, math.nan)):
        t[~mask] = bad
    pat = [ops.DENSE] * H
    out, lse, rest = ops.frame_attn_fwd(q, k, v, pat, token_mask=mask, rest=True)
    grads = ops.frame_attn_bwd(do, q, k, v, out, lse, pat, token_mask=mask, rest=rest)
    for t in (out, *grads):
        assert (t[~mask] == 0).all()
    assert (lse.transpose(1, 2)[~mask] == -math.inf).all()
    for h in sorted({0, H - 1}):
        Q, K, V, G = (t[0, mask[0], h].double() for t in (q, k, v, do))
        s = Q @ K.t().contiguous() * 0.125
        L = torch.logsumexp(s, -1)
        p = torch.exp(s - L[:, None])
        o = p @ V
        ds = p * (G @ V.t().contiguous() - (G * o).sum(-1, keepdim=True)) * 0.125
        assert (lse[0, h, mask[0]].double() - L).abs().max() < 1e-5 * L.abs().max()
        for name, t, w in (("out", out, o), ("dq", grads[0], ds @ K), ("dk", grads[1], ds.t().contiguous() @ Q),
                           ("dv", grads[2], p.t().contiguous() @ G)):
            rel = float((t[0, mask[0], h].double() - w).norm() / w.norm())
            # a result's rounding and its operands' (P, dS, D), each at most U of magnitudes that add in quadrature
            assert rel < 2 * R.U, (name, h, rel)


@pytest.mark.parametrize("pattern,B,F,T,H", [("mix", 1, 2, 40, 64), ("mix", 1, 300, 1, 5), ("anchor_local", 2, 50, 7, 3),
                                             ("mix", 5, 1, 1, 64)])
def test_many_heads_and_small_frames(ops, pattern, B, F, T, H):
    q, k, v, do = inputs(B, F * T, H, H + T)
    check(ops, q, k, v, do, patterns_of(ops, pattern, H), F)


def test_one_tensor_for_all_and_broadcast_gradient(ops):
    """q, k and v are one tensor; dout is one row for all tokens, read in place."""
    B, N, H = 2, 200, 3
    x = inputs(B, N, H, 21)[0]
    do = inputs(B, N, H, 22)[3][:, :1, :, :]
    pat = patterns_of(ops, "mix", H)
    want = check(ops, x, x, x, do.expand(B, N, H, 64), pat, 2)
    gx, gdo = x.to(DEV), do.to(DEV).expand(B, N, H, 64)
    out, lse, rest = ops.frame_attn_fwd(gx, gx, gx, pat, frames=2, rest=True)
    for n, t in zip(("dq", "dk", "dv"), ops.frame_attn_bwd(gdo, gx, gx, gx, out, lse, pat, frames=2, rest=rest)):
        assert torch.equal(t, want[n]), n
    bad = torch.empty(B, 1, H, 64, dtype=torch.bfloat16, device=DEV).expand(B, N, H, 64)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.frame_attn_bwd(gdo, gx, gx, gx, out, lse, pat, frames=2, rest=rest, grads=(bad, *want_like(gx, 2)))


def want_like(t, n):
    return [torch.empty_like(t) for _ in range(n)]


@pytest.mark.parametrize("B,F,T,H", [(1, 1, 900, 2), (2, 2, 300, 14), (1, 1, 2060, 16)])
def test_shared_walks_captured(ops, B, F, T, H):
    """Launches that share their walks in a graph whose inputs and mask change between the replays."""
    N = F * T
    pat = [ops.DENSE] * H
    gen = torch.Generator().manual_seed(T)
    bufs = [t.to(DEV) for t in inputs(B, N, H, 1)]
    mask = torch.ones(B, N, dtype=torch.bool, device=DEV)

    def run():
        res = []
        for m in (None, mask):
            out, lse, rest = ops.frame_attn_fwd(*bufs[:3], pat, frames=F, token_mask=m, rest=True)
            res += [out, lse, *ops.frame_attn_bwd(bufs[3], *bufs[:3], out, lse, pat, frames=F, token_mask=m, rest=rest)]
        return res
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for seed in (3, 4, 5):
        for dst, src in zip(bufs, inputs(B, N, H, seed)):
            dst.copy_(src)
        mask.copy_(torch.rand(B, N, generator=gen) < 0.3 * (seed - 2))
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got)), seed
