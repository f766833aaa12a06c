"""The block's operators as a training step uses them: ``autograd.linear``, ``autograd.residual_norm`` and
``autograd.dropout`` in a chain, a transformer block and a model with "saf3r_block", patched layers with
``linear_kernels``; against the same in 64 bits with the same masks."""
import importlib
import math
import threading

import pytest
import torch
import torch.utils.checkpoint
import torch.nn.functional as F

import block_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF, FP = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def mods(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return [importlib.import_module(pkg.__name__ + m) for m in (".autograd", ".ops", ".aggregator", ".patch", ".vggt")]


def rel(a, b):
    return float((a.double().cpu() - b.double().cpu()).norm() / b.double().cpu().norm())


def leaves(*ts):
    return [t.detach().to(DEV).requires_grad_() for t in ts]


@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("dt", [BF, FP])
def test_functions_in_a_chain(mods, dt, master):
    """residual_norm -> linear (GELU, dropout) -> linear (gate, residual) -> dropout, with 16-bit or fp32 parameters."""
    ad = mods[0]
    g = torch.Generator().manual_seed(0)

    def rnd(*shape, scale=1.0, kind=dt):
        return (scale * torch.randn(*shape, generator=g)).to(kind)
    pk = F32 if master else dt
    x, branch = rnd(3, 50, 96, kind=pk), rnd(3, 50, 96)
    params = [rnd(96, scale=0.5, kind=pk), 1 + rnd(96, scale=0.2, kind=pk), rnd(96, scale=0.1, kind=pk),
              rnd(200, 96, scale=0.1, kind=pk), rnd(200, scale=0.1, kind=pk),
              rnd(96, 200, scale=0.07, kind=pk), rnd(96, scale=0.1, kind=pk), rnd(96, scale=0.5, kind=pk)]
    states = [torch.randint(-(1 << 62), 1 << 62, (2,), generator=g) for _ in range(3)]
    p = [0.1, 0.25, 0.5]
    got = leaves(x, branch, *params)
    st = [s.to(DEV) for s in states]
    h, y = ad.residual_norm(got[0], got[1], got[2], got[3], got[4], 1e-5, p[0], st[0])
    u = ad.linear(y, got[5], got[6], "gelu", dropout=p[1], state=st[1])
    z = ad.linear(u, got[7], got[8], gate=got[9], residual=h)
    out = ad.dropout(z, p[2], state=st[2])
    dout = rnd(*out.shape, scale=0.1, kind=out.dtype)
    out.backward(dout.to(DEV))
    want = [t.double().requires_grad_() for t in (x, branch, *params)]
    f = [R.keep_factor(a, s, 150, n).reshape(3, 50, n) for a, s, n in zip(p, states, (96, 200, 96))]
    h = want[0] + want[2] * f[0] * want[1]
    y = F.layer_norm(h, (96,), want[3], want[4], 1e-5)
    u = F.gelu(F.linear(y, want[5], want[6])) * f[1]
    z = h + want[9] * F.linear(u, want[7], want[8])
    ref = z * f[2]
    ref.backward(dout.double())
    # independent roundings to 16 bits: h, y, kept, u, z, out forward; as many gradients backward; the parameters
    tol = R.half_step(dt) * 20 ** 0.5
    assert out.dtype == pk and rel(out, ref.detach()) < tol
    for i, (a, b, t) in enumerate(zip(got, want, (x, branch, *params))):
        assert a.grad.dtype == t.dtype and rel(a.grad, b.grad) < tol, (i, rel(a.grad, b.grad))


def test_new_masks_and_repeated_ones(mods):
    """Every call draws its mask; one seed repeats them; forward and backward of a call share it."""
    ad = mods[0]
    x, w = leaves(torch.randn(64, 64).to(BF), torch.eye(64).to(BF))
    torch.manual_seed(5)
    a, b = ad.linear(x, w, dropout=0.5), ad.linear(x, w, dropout=0.5)
    torch.manual_seed(5)
    assert torch.equal(ad.linear(x, w, dropout=0.5), a) and not torch.equal(a, b)
    (dx,) = torch.autograd.grad(a, x, torch.ones_like(a))
    assert torch.equal(dx != 0, a != 0)
    y = ad.dropout(x, 0.5)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(dx != 0, y != 0) and float(dx.max()) == 2.0
    assert ad.dropout(x, 0.5, training=False) is x and ad.dropout(x, 0.0) is x


def test_without_gradients_and_twice(mods):
    ad = mods[0]
    x, w = torch.randn(8, 64, device=DEV).to(BF), torch.randn(64, 64, device=DEV).to(BF)
    assert not ad.linear(x, w, activation="gelu").requires_grad
    xg, wg = leaves(x, w)
    y = ad.linear(xg, w, activation="gelu")
    y.sum().backward()
    assert xg.grad is not None
    (dx,) = torch.autograd.grad(ad.linear(xg, wg).sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    h, z = ad.residual_norm(xg, x)
    (dx,) = torch.autograd.grad(h.sum(), xg)  # (the norm's result is not used)
    assert torch.equal(dx, torch.ones_like(dx))
    h, z = ad.residual_norm(xg, x)
    (dz,) = torch.autograd.grad(z.float().square().sum(), xg)
    assert torch.isfinite(dz).all()


def grid(S, gh, gw, ns):
    yy, xx = torch.meshgrid(torch.arange(gh), torch.arange(gw), indexing="ij")
    patch = torch.stack([yy.flatten(), xx.flatten()], -1) + 1
    return torch.cat([torch.zeros(ns, 2, dtype=torch.long), patch])[None].expand(S, -1, -1).contiguous()


@pytest.mark.parametrize("drop", [0.0, 0.2])
@pytest.mark.parametrize("mode", ["bf16", "autocast"])
def test_block(mods, monkeypatch, mode, drop):
    """A block's step against torch's operators in 64 bits with the same masks."""
    ad, ops, agg, _, _ = mods
    torch.manual_seed(1)
    block = agg.Block(256, 4, 4.0, 0.5, True, agg.RotaryPositionEmbedding2D(100.0), drop=drop)
    for q in (block.ls1.gamma, block.ls2.gamma):
        torch.nn.init.uniform_(q, 0.5, 1.0)
    if mode == "bf16":
        block = block.to(BF)
    ref = agg.Block(256, 4, 4.0, 0.5, True, agg.RotaryPositionEmbedding2D(100.0)).double()
    ref.load_state_dict(block.state_dict())
    drawn = []

    def state(device="cuda"):
        drawn.append(torch.tensor([77 + len(drawn), 3], dtype=torch.int64))
        return drawn[-1].to(device)
    monkeypatch.setattr(ops, "dropout_state", state)
    block = block.to(DEV)
    block.frame_attention = "saf3r_block"
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 47, 256, generator=g)
    x = x.to(BF) if mode == "bf16" else x
    pos = grid(2, 6, 7, 5)
    xg = x.to(DEV).requires_grad_()
    with torch.autocast("cuda", dtype=BF, enabled=mode == "autocast"):
        out = block(xg, pos=pos.to(DEV), positions=8)
    dout = (0.1 * torch.randn(out.shape, generator=g)).to(out.dtype)
    out.backward(dout.to(DEV))
    assert out.dtype == x.dtype and len(drawn) == (3 if drop else 0)
    keep = [R.keep_factor(drop, s, 94, n).reshape(2, 47, n) for s, n in zip(drawn, (256, 1024, 256))] or [1.0] * 3
    xr = x.double().requires_grad_()
    h = xr + ref.ls1(ref.attn(ref.norm1(xr), pos=pos) * keep[0])
    m = ref.mlp
    want = h + ref.ls2(m.fc2(m.act(m.fc1(ref.norm2(h))) * keep[1]) * keep[2])
    want.backward(dout.double())
    # twelve roundings to bf16 on the way and as many back (two norms, qkv, head norm, attention, projection, the stream
    # twice, z, u, the products' gradients), each of independent errors
    tol = 2 * R.half_step(BF) * 24 ** 0.5
    assert rel(out, want.detach()) < tol and rel(xg.grad, xr.grad) < tol
    theirs = dict(ref.named_parameters())
    off = sum(float((p.grad.double().cpu() - theirs[n].grad).norm() ** 2) for n, p in block.named_parameters())
    total = sum(float(p.grad.norm() ** 2) for p in theirs.values())
    assert math.sqrt(off / total) < tol
    for n, p in block.named_parameters():
        assert torch.isfinite(p.grad).all() and p.grad.dtype == p.dtype, n


@pytest.mark.parametrize("autocast", [False, True])
def test_model(mods, autocast):
    """A step of the aggregator with "saf3r_block", one global layer patched with ``linear_kernels``: as with
    "saf3r_train" up to the roundings, and its inference as its training's forward."""
    ad, ops, agg, patch, _ = mods

    def build(kind):
        torch.manual_seed(0)
        m = agg.VGGTAggregatorModel(img_size=84, embed_dim=256, depth=2, num_heads=4, dino_depth=1, dino_dim=256,
                                    dino_heads=4, frame_attention=kind)
        for b in list(m.aggregator.global_blocks) + list(m.aggregator.frame_blocks):
            torch.nn.init.uniform_(b.ls1.gamma, 0.5, 1.0)
            torch.nn.init.uniform_(b.ls2.gamma, 0.5, 1.0)
        m = m.to(DEV) if autocast else m.to(DEV).to(BF)
        patch.patch_model(m, "vggt", {"patch_module": {"type": "headsparse", "trainable": True,
                                                       "linear_kernels": kind == "saf3r_block"}, "sparse_config": {"0": []}})
        patch.update_args_per_forward(m, "vggt", 84, 84)
        return m
    images = agg.blurred_frames(3, size=84, sigma=1.5, seed=3).to(DEV)
    images = images if autocast else images.to(BF)
    res = {}
    for kind in ("saf3r_train", "saf3r_block"):
        m = build(kind)
        with torch.autocast("cuda", dtype=BF, enabled=autocast):
            out = m(images)[0][-1]
            g = torch.Generator().manual_seed(2)
            out.backward((0.1 * torch.randn(out.shape, generator=g)).to(DEV).to(out.dtype))
            with torch.no_grad():
                again = m(images)[0][-1]
        # (without gradients the patched layer runs through the packed kernels: other roundings)
        assert rel(again, out.detach()) < 2 * R.half_step(BF) * 100 ** 0.5
        res[kind] = out.detach(), {n: p.grad for n, p in m.named_parameters()}
    (a, ga), (b, gb) = res.values()
    tol = 2 * R.half_step(BF) * (2 * 5 * 20) ** 0.5  # five blocks of about twenty roundings each way, on both sides
    assert a.dtype == b.dtype and rel(b, a) < tol
    off = total = 0.0
    for n, p in ga.items():
        assert (p is None) == (gb[n] is None), n
        if p is not None:
            off += float((p.double() - gb[n].double()).norm() ** 2)
            total += float(p.double().norm() ** 2)
    assert math.sqrt(off / total) < tol


def test_block_in_a_graph(mods):
    """A captured step draws new masks in every replay and gives the eager step's gradients for the same seeds."""
    ad, ops, agg, _, _ = mods
    torch.manual_seed(1)
    block = agg.Block(128, 2, 2.0, 0.5, drop=0.3).to(BF).to(DEV)
    block.frame_attention = "saf3r_block"
    x = torch.randn(1, 70, 128, device=DEV).to(BF)
    dout = torch.randn(1, 70, 128, device=DEV).to(BF)
    params = list(block.parameters())

    def step():
        return block(x).detach(), torch.autograd.grad(block(x), params, dout)  # (no graph of the leaves outlives a step)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    seen = []
    for seed in range(3):
        torch.manual_seed(seed)
        graph.replay()
        torch.cuda.synchronize()
        seen.append(held[0].clone())
        got = [t.clone() for t in held[1]]
        torch.manual_seed(seed)
        out, want = step()
        assert torch.equal(seen[-1], out)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_no_rows_with_gradients(mods):
    ad, ops, _, _, _ = mods
    w, b, g = (torch.randn(*s, device=DEV).to(BF).requires_grad_() for s in ((72, 64), (72,), (72,)))
    x = torch.zeros(0, 64, device=DEV, dtype=BF, requires_grad=True)
    ad.linear(x, w, b, "gelu", g, dropout=0.3).sum().backward()
    assert x.grad.shape == x.shape and all(not t.grad.any() for t in (w, b, g))
    stream = torch.zeros(0, 3, 72, device=DEV, requires_grad=True)
    g.grad = None
    h, y = ad.residual_norm(stream, torch.zeros(0, 3, 72, device=DEV, dtype=BF), g, dropout=0.3)
    (h.sum() + y.sum()).backward()
    assert h.shape == stream.grad.shape and not g.grad.any()
    z = torch.zeros(0, 5, device=DEV, requires_grad=True)
    ad.dropout(z, 0.5).sum().backward()
    assert z.grad.shape == z.shape


def test_one_weight_twice_and_the_rows_as_residual(mods):
    ad, ops, _, _, _ = mods
    g = torch.Generator().manual_seed(7)
    w = (torch.randn(64, 64, generator=g) / 8).to(BF).to(DEV).requires_grad_()
    x = torch.randn(50, 64, generator=g).to(BF).to(DEV).requires_grad_()
    dy = torch.randn(50, 64, generator=g).to(BF).to(DEV)
    y = ad.linear(ad.linear(x, w, residual=x), w, activation="gelu")
    y.backward(dy)
    w2, x2 = (t.detach().double().requires_grad_() for t in (w, x))
    want = torch.nn.functional.gelu((x2 @ w2.t() + x2) @ w2.t())
    want.backward(dy.double())
    tol = 2 * R.half_step(BF) * 7 ** 0.5  # seven roundings at most, forward and backward, each of a value's own size or less
    assert rel(y, want) < tol and rel(x.grad, x2.grad) < tol and rel(w.grad, w2.grad) < tol


def test_two_graphs_and_two_threads(mods):
    """Graphs that are replayed on two streams at a time, and threads that call at a time, have workspaces of their own."""
    _, ops, _, _, _ = mods
    g = torch.Generator().manual_seed(8)
    w, b, gate = ((torch.randn(*s, generator=g) / 8).to(BF).to(DEV) for s in ((72, 1032), (72,), (72,)))
    xs = [torch.randn(300, 1032, generator=g).to(BF).to(DEV) for _ in range(2)]
    dys = [torch.randn(300, 72, generator=g).to(BF).to(DEV) for _ in range(2)]
    state = torch.tensor([3, 4], device=DEV)

    def step(i):
        y, kept = ops.linear_fwd(xs[i], w, b, "gelu", gate, dropout=0.2, state=state, keep=True)
        return (y, *ops.linear_bwd(dys[i], xs[i], w, kept, "gelu", gate, 0.2, state))
    want = [[t.clone() for t in step(i)] for i in range(2)]
    torch.cuda.synchronize()
    graphs, held = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            held.append(step(i))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(held[i], want[i]))
    same = {}

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(5):
                res = step(i)
            streams[i].synchronize()
            same[i] = all(torch.equal(a, b) for a, b in zip(res, want[i]))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert same == {0: True, 1: True}


def test_checkpointed_block(mods):
    """A block that is computed again in its backward pass drops the same elements again."""
    ad, ops, agg, _, _ = mods
    torch.manual_seed(1)
    block = agg.Block(128, 2, 2.0, 0.5, drop=0.3).to(BF).to(DEV)
    block.frame_attention = "saf3r_block"
    x = torch.randn(2, 70, 128, device=DEV).to(BF).requires_grad_()
    dout = torch.randn(2, 70, 128, device=DEV).to(BF)
    res = []
    for again in (False, True):
        torch.manual_seed(3)
        y = torch.utils.checkpoint.checkpoint(block, x, use_reentrant=False) if again else block(x)
        res.append((y.detach(), *torch.autograd.grad(y, [x, *block.parameters()], dout)))
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_patched_layer(mods):
    """``linear_kernels`` of a patched layer against its torch products."""
    ad, ops, agg, patch, vggt = mods
    res = []
    for on in (False, True):
        torch.manual_seed(0)
        model = vggt.GlobalAttentionStack(1, 256, 4).to(BF).to(DEV)
        patch.patch_model(model, "vggt", {"patch_module": {"type": "headsparse", "trainable": True, "linear_kernels": on},
                                          "sparse_config": {"0": [{"mode": "global_to_frame", "head_ids": [1]}]}})
        patch.update_args_per_forward(model, "vggt", 84, 98)
        attn = model.aggregator.global_blocks[0].attn
        g = torch.Generator().manual_seed(4)
        x = torch.randn(1, 2 * 47, 256, generator=g).to(BF).to(DEV).requires_grad_()
        out = attn(x, grid(2, 6, 7, 5).reshape(1, -1, 2).to(DEV))
        out.backward(torch.randn(out.shape, generator=g).to(BF).to(DEV))
        res.append((out.detach(), x.grad, *(p.grad for p in attn.parameters())))
    tol = 2 * R.half_step(BF) * 14 ** 0.5  # six or seven roundings each way on both sides
    for a, b in zip(*res):
        assert rel(b, a) < tol


def test_other_current_stream_and_concurrent_calls(mods):
    """Two streams at once, each with its own workspaces and masks."""
    ad, ops = mods[:2]
    x = torch.randn(1041, 1024, device=DEV).to(BF)
    w = torch.randn(512, 1024, device=DEV).to(BF) / 32
    st = torch.tensor([1, 2], device=DEV)
    dy = torch.randn(1041, 512, device=DEV).to(BF)

    def step(scale):
        y, kept = ops.linear_fwd(x * scale, w, activation="gelu", dropout=0.1, state=st, keep=True)
        return (y, *ops.linear_bwd(dy, x * scale, w, kept, "gelu", dropout=0.1, state=st)[:3])
    want = [step(1.0), step(2.0)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        got = []
        for s, scale in zip(streams, (1.0, 2.0)):
            with torch.cuda.stream(s):
                got.append(step(scale))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
