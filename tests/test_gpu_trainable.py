"""Training through the kernels: the differentiable functions, the patched layer with ``trainable``, and a model's step,
against torch's differentiation of the same formulas in 64 bits."""
import importlib

import pytest
import torch

import train_ref as R
from oracle import attention as OA

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def mods(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return tuple(importlib.import_module(pkg.__name__ + m) for m in (".autograd", ".ops", ".patch", ".aggregator", ".vggt"))


def rel(a, b):
    return float((a.detach().double().cpu() - b).norm() / b.norm())


def layer64(x, pos, params, patterns, frames, heads, eps, base=100.0):
    """A patched attention layer of x [1, N, C] in 64 bits: qkv, norms, rotary positions, attention, projection."""
    B, N, C = x.shape
    qkv = (x @ params["qkv.weight"].T + params["qkv.bias"]).reshape(B, N, 3, heads, 64)
    q, k, v = qkv.unbind(2)
    q = R.layer_norm(q, params["q_norm.weight"], params["q_norm.bias"], eps)[0]
    k = R.layer_norm(k, params["k_norm.weight"], params["k_norm.bias"], eps)[0]
    ang = torch.arange(int(pos.max()) + 1, dtype=torch.float64)[:, None] * base ** -(torch.arange(0, 32, 2) / 32)
    parts = []
    for t in (q, k):
        halves = []
        for a in range(2):
            c, s = ang.cos()[pos[..., a]][:, :, None], ang.sin()[pos[..., a]][:, :, None]
            u, w = t[..., 32 * a:32 * a + 16], t[..., 32 * a + 16:32 * a + 32]
            halves += [u * c - w * s, w * c + u * s]
        parts.append(torch.cat(halves, -1))
    q, k = parts
    geom = OA.Geometry(frames, N // frames, 0)
    outs = []
    for h in range(heads):
        if patterns[h] == OA.SKIP:
            outs.append(torch.zeros(B, N, 64, dtype=torch.float64))
            continue
        ok = OA.allowed_mask(patterns[h], torch.arange(N), geom)
        s = (q[:, :, h] @ k[:, :, h].transpose(1, 2) * 0.125).masked_fill(~ok, -float("inf"))
        outs.append(torch.softmax(s, -1) @ v[:, :, h])
    return torch.cat(outs, -1) @ params["proj.weight"].T + params["proj.bias"]


def grid_positions(frames, ph, pw, special):
    yy, xx = torch.meshgrid(torch.arange(ph), torch.arange(pw), indexing="ij")
    patch = torch.stack([yy.flatten(), xx.flatten()], -1) + 1
    return torch.cat([torch.zeros(special, 2, dtype=torch.long), patch]).repeat(frames, 1)[None]


GROUPS = [{"mode": "full", "head_ids": [0]}, {"mode": "global_to_frame", "head_ids": [1]},
          {"mode": "anchor_local", "head_ids": [2]}, {"mode": "all_to_first", "head_ids": [3]},
          {"mode": "skip", "head_ids": [4]}]


def patched(mods, ph, pw, dtype, groups=GROUPS, heads=5, trainable=True):
    _, _, patch, _, vggt = mods
    torch.manual_seed(3)
    model = vggt.GlobalAttentionStack(depth=1, dim=64 * heads, num_heads=heads)
    attn = model.aggregator.global_blocks[0].attn
    for n in (attn.q_norm, attn.k_norm):
        torch.nn.init.uniform_(n.weight, 0.5, 1.5)
        torch.nn.init.normal_(n.bias, std=0.2)
    model = model.to(DEV).to(dtype)
    patch.patch_model(model, "vggt", {"patch_module": {"type": "headsparse", "trainable": trainable},
                                      "sparse_config": {"0": groups}})
    patch.update_args_per_forward(model, "vggt", 14 * ph, 14 * pw)
    return model.aggregator.global_blocks[0].attn


@pytest.mark.parametrize("frames,ph,pw,dtype,autocast", [(3, 6, 7, BF, False), (1, 5, 5, BF, False),
                                                         (2, 9, 8, torch.float32, True)])
def test_patched_layer_gradients(mods, frames, ph, pw, dtype, autocast):
    _, ops, _, _, _ = mods
    w = patched(mods, ph, pw, dtype)
    N = frames * (5 + ph * pw)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, N, 320, generator=g).to(dtype)
    dy = (0.1 * torch.randn(1, N, 320, generator=g)).to(dtype)
    pos = grid_positions(frames, ph, pw, 5)
    gx = x.to(DEV).requires_grad_()
    with torch.autocast("cuda", dtype=BF, enabled=autocast):
        y = w(gx, pos.to(DEV))
        with torch.no_grad():
            packed = w(gx, pos.to(DEV))
    y.backward(dy.to(DEV).to(y.dtype))
    names = ("qkv.weight", "qkv.bias", "q_norm.weight", "q_norm.bias", "k_norm.weight", "k_norm.bias", "proj.weight",
             "proj.bias")
    got = dict(w.orig_module.named_parameters())
    params = {n: got[n].detach().double().cpu().requires_grad_() for n in names}
    x64 = x.double().requires_grad_()
    y64 = layer64(x64, pos, params, w.patterns, frames, 5, w.orig_module.q_norm.eps)
    y64.backward(dy.double())
    # bf16 roundings on the way (x and weights under autocast, qkv, the rotated rows, P, the output, and backwards dout,
    # dS, dq/dk/dv, dqkv, the result): at most ten of half a step each, were they all to add up
    tol = 10 * R.U
    assert rel(y, y64.detach()) < tol and rel(packed, y64.detach()) < tol
    assert rel(gx.grad, x64.grad) < tol
    for n in names:
        if n == "k_norm.bias" or n == "qkv.bias":  # (a shift of all keys changes no softmax of a row without rotation)
            assert (got[n].grad.double().cpu() - params[n].grad).norm() < tol * params["q_norm.bias"].grad.norm() + \
                tol * params[n].grad.norm(), n
        else:
            assert rel(got[n].grad, params[n].grad) < tol, (n, rel(got[n].grad, params[n].grad))


def test_trainable_is_asked_for(mods):
    """Without ``trainable``, and where no gradient is needed, the packed path runs as before; heads that have no
    gradients are refused when the model is patched."""
    _, ops, patch, _, vggt = mods
    w = patched(mods, 6, 7, BF)
    x = torch.randn(1, 3 * 47, 320, generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    pos = grid_positions(3, 6, 7, 5).to(DEV)
    plain = patched(mods, 6, 7, BF, trainable=False)
    with torch.no_grad():
        a, b = w(x, pos), plain(x, pos)
    assert torch.equal(a, b)
    for p in w.parameters():
        p.requires_grad_(False)
    assert torch.equal(w(x, pos), a)
    for mode in ({"mode": "stride", "stride": 4}, {"mode": "block_topk"}, {"mode": "broadcast_first"}):
        with pytest.raises(NotImplementedError, match=mode["mode"]):
            patched(mods, 6, 7, BF, [{**mode, "head_ids": [1]}])


@pytest.mark.parametrize("autocast", [False, True])
def test_training_step_of_a_model(mods, autocast):
    """A step of the aggregator with every block's norms and attention through the kernels, its global layers patched:
    every parameter's gradient close to that of the same model in fp32 on torch's operators."""
    _, ops, patch, agg, _ = mods
    def build(kind):
        torch.manual_seed(0)
        m = agg.VGGTAggregatorModel(img_size=14 * 6, embed_dim=256, depth=2, num_heads=4, dino_depth=1, dino_dim=256,
                                    dino_heads=4, frame_attention=kind)
        for b in list(m.aggregator.global_blocks) + list(m.aggregator.frame_blocks):
            torch.nn.init.uniform_(b.ls1.gamma, 0.5, 1.0)
        return m
    images = agg.blurred_frames(3, size=84, sigma=1.5, seed=3)
    ref = build("sdpa").double()
    ref_out = ref(images.double())[0]
    g = torch.Generator().manual_seed(2)
    dy = 0.1 * torch.randn(ref_out[-1].shape, generator=g, dtype=torch.float64)
    ref_out[-1].backward(dy)
    m = build("saf3r_train").to(DEV)
    if not autocast:
        m = m.to(BF)
    cfg = {"patch_module": {"type": "headsparse", "trainable": True}, "sparse_config": {"0": []}}  # layer 1: unpatched
    patch.patch_model(m, "vggt", cfg)
    patch.update_args_per_forward(m, "vggt", 84, 84)
    with torch.autocast("cuda", dtype=BF, enabled=autocast):
        out = m(images.to(DEV) if autocast else images.to(DEV).to(BF))[0][-1]
    out.backward(dy.to(DEV).to(out.dtype))
    # five blocks of about twenty bf16 roundings each way, adding up as independent errors
    tol = R.U * (2 * 5 * 20) ** 0.5
    assert rel(out, ref_out[-1].detach()) < tol
    want = dict(ref.named_parameters())
    total = sum(float(p.grad.norm() ** 2) for p in want.values() if p.grad is not None) ** 0.5
    off = 0.0
    for n, p in m.named_parameters():
        key = n.replace(".orig_module", "")
        if want[key].grad is None:
            assert p.grad is None
            continue
        assert torch.isfinite(p.grad).all(), n
        off += float((p.grad.double().cpu() - want[key].grad).norm() ** 2)
    assert off ** 0.5 < tol * total, off ** 0.5 / total


def test_functions_against_64_bits(mods):
    """layer_norm -> head_rotary -> frame_attention in a chain, with broadcast and shared inputs."""
    ad, ops, _, _, _ = mods
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 40, 1, 3, 64, generator=g).to(BF)
    w = (1 + 0.2 * torch.randn(1, 64, generator=g))
    b = 0.1 * torch.randn(1, 64, generator=g)
    kshared = torch.randn(1, 40, 1, 64, generator=g).to(BF)  # one head's rows of one clip, broadcast to all
    pos = torch.randint(0, 20, (2, 40, 1), generator=g)
    cos, sin = ops.rotary_tables(20, 64, device="cpu")
    do = torch.randn(2, 40, 3, 64, generator=g).to(BF)
    gx, gw, gb, gk = (t.to(DEV).requires_grad_() for t in (x, w, b, kshared))
    q = ad.head_rotary(gx, pos.to(DEV), (cos.to(DEV), sin.to(DEV)), norm=True, weight=gw, bias=gb)[:, :, 0]
    kk = gk.expand(2, 40, 3, 64)
    out = ad.frame_attention(q, kk, kk, [ops.DENSE, ops.FRAME_LOCAL, ops.ANCHOR], frames=2)
    out.backward(do.to(DEV))
    x64, w64, b64, k64 = (t.double().requires_grad_() for t in (x, w, b, kshared))
    y = R.rotate(R.layer_norm(x64, w64[:, None], b64[:, None], 1e-5)[0], pos, cos, sin, "half", 64)[:, :, 0]
    outs = []
    geom = OA.Geometry(2, 20, 0)
    for h, p in enumerate((OA.DENSE, OA.FRAME_LOCAL, OA.ANCHOR)):
        ok = OA.allowed_mask(p, torch.arange(40), geom)
        kh = k64[:, :, 0].expand(2, 40, 64)
        outs.append(torch.softmax((y[:, :, h] @ kh.transpose(1, 2) * 0.125).masked_fill(~ok, -float("inf")), -1) @ kh)
    ref = torch.stack(outs, 2)
    ref.backward(do.double())
    tol = 8 * R.U  # rotated rows, P, out, dS, dq / dk / dv, dx
    assert rel(out, ref.detach()) < tol
    for a, r in ((gx, x64), (gw, w64), (gb, b64), (gk, k64)):
        assert a.grad.shape == r.grad.shape and rel(a.grad, r.grad) < tol
    n = torch.randn(7, 96, device=DEV, requires_grad=True)
    z = ad.layer_norm(n, None, None, 1e-5, BF)
    assert z.dtype == BF
    (gn,) = torch.autograd.grad(z.float().square().sum(), n, create_graph=False)
    assert gn.shape == n.shape
    with pytest.raises(RuntimeError):
        (gn,) = torch.autograd.grad(ad.layer_norm(n).square().sum(), n, create_graph=True)
        gn.sum().backward()


def test_frozen_inputs(mods):
    """Only what needs a gradient gets one."""
    ad, ops, _, _, _ = mods
    q, k, v = (torch.randn(1, 30, 2, 64, device=DEV).to(BF) for _ in range(3))
    assert not ad.frame_attention(q, k, v, [0, 0]).requires_grad
    v.requires_grad_()
    ad.frame_attention(q, k, v, [0, 0]).sum().backward()
    assert v.grad is not None and q.grad is None
    x = torch.randn(5, 64, device=DEV)
    w = torch.ones(64, device=DEV, requires_grad=True)
    ad.layer_norm(x, w, torch.zeros(64, device=DEV)).sum().backward()
    assert w.grad.shape == (64,) and x.grad is None


def test_captured_training_step(mods):
    """Forward and backward of the whole layer in one graph, replayed on new inputs between eager steps."""
    ad, ops, _, _, _ = mods
    patterns = [ops.DENSE, ops.FRAME_LOCAL, ops.ANCHOR_LOCAL, ops.ANCHOR]
    pos = grid_positions(2, 6, 7, 5).to(DEV)
    tables = ops.rope_tables(10, 100.0, DEV)
    N = pos.shape[1]
    qkv = torch.randn(1, N, 3 * 256, device=DEV).to(BF).requires_grad_()
    w = torch.rand(2, 64, device=DEV).add_(0.5).requires_grad_()
    b = torch.randn(2, 64, device=DEV).requires_grad_()
    dy = torch.randn(1, N, 256, device=DEV).to(BF)

    def step():
        y = ad.qkv_attention(qkv, patterns, 2, pos, tables, True, w, b)
        return (y.detach(), *torch.autograd.grad(y, (qkv, w, b), dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        with torch.no_grad():
            qkv.copy_(torch.randn(1, N, 768, generator=g))
            dy.copy_(torch.randn(1, N, 256, generator=g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, held)), seed


def test_qkv_attention_without_prologue(mods):
    ad, ops, _, _, _ = mods
    qkv = torch.randn(2, 50, 3 * 128, device=DEV).to(BF).requires_grad_()
    y = ad.qkv_attention(qkv, [ops.DENSE, ops.SKIP])
    y.backward(torch.ones_like(y).expand_as(y))
    x = qkv.detach().view(2, 50, 3, 2, 64)
    leaves = [x[:, :, i].clone().requires_grad_() for i in range(3)]
    ad.frame_attention(*leaves, [ops.DENSE, ops.SKIP]).backward(torch.ones(2, 50, 2, 64, device=DEV, dtype=BF))
    assert torch.equal(qkv.grad.view(x.shape), torch.stack([t.grad for t in leaves], 2))
    with pytest.raises(ValueError, match="qkv must be"):
        ad.qkv_attention(qkv, [ops.DENSE])


def test_argument_checks(mods):
    _, ops, _, _, _ = mods
    t = torch.zeros(1, 6, 2, 64, dtype=BF, device=DEV)
    lse = torch.zeros(1, 2, 6, device=DEV)
    bad = [
        ("q must be", lambda: ops.frame_attn_fwd(t[..., :32], t, t, [0, 0])),
        ("k must have", lambda: ops.frame_attn_fwd(t, t[:, :5], t, [0, 0])),
        ("bfloat16", lambda: ops.frame_attn_fwd(t.float(), t.float(), t.float(), [0, 0])),
        ("frames of one size", lambda: ops.frame_attn_fwd(t, t, t, [0, 0], frames=4)),
        ("frames of one size", lambda: ops.frame_attn_fwd(t, t, t, [0, 0], frames=0)),
        ("one pattern per head", lambda: ops.frame_attn_fwd(t, t, t, [0])),
        ("token_mask", lambda: ops.frame_attn_fwd(t, t, t, [0, 0], token_mask=torch.ones(1, 5, device=DEV).bool())),
        ("token_mask", lambda: ops.frame_attn_fwd(t, t, t, [0, 0], token_mask=torch.ones(1, 6, device=DEV))),
        ("GPU", lambda: ops.frame_attn_fwd(t, t, t, [0, 0], token_mask=torch.ones(1, 6).bool())),
        ("dout must be", lambda: ops.frame_attn_bwd(t[:, :5], t, t, t, t, lse, [0, 0])),
        ("out must be", lambda: ops.frame_attn_bwd(t, t, t, t, t.float(), lse, [0, 0])),
        ("lse must be", lambda: ops.frame_attn_bwd(t, t, t, t, t, lse[:, :1], [0, 0])),
        ("rest must be", lambda: ops.frame_attn_bwd(t, t, t, t, t, lse, [0, 0], rest=t.float())),
        ("grads", lambda: ops.frame_attn_bwd(t, t, t, t, t, lse, [0, 0], grads=(t, t, t.float()))),
        ("grads need", lambda: ops.frame_attn_bwd(t, t, t, t, t, lse, [0, 0], grads=(
            t.clone(), t.clone(), torch.zeros(1, 6, 2, 65, dtype=BF, device=DEV)[..., :64]))),
        ("x must be", lambda: ops.head_rotary_fwd(t, norm=True)),
        ("neither", lambda: ops.head_rotary_fwd(t[:, :, None])),
        ("layout", lambda: ops.head_rotary_fwd(t[:, :, None], norm=True, layout="other")),
        ("belong to the norm", lambda: ops.head_rotary_fwd(t[:, :, None], torch.zeros(1, 6, 1, device=DEV).long(),
                                                            ops.rotary_tables(3, 64, device=DEV),
                                                            weight=torch.ones(1, 64, device=DEV))),
        ("pos and tables", lambda: ops.head_rotary_fwd(t[:, :, None], norm=True, tables=ops.rotary_tables(3, 64))),
        ("pos must be", lambda: ops.head_rotary_fwd(t[:, :, None], torch.zeros(1, 6, device=DEV).long(),
                                                    ops.rotary_tables(3, 64, device=DEV))),
        ("int32 or int64", lambda: ops.head_rotary_fwd(t[:, :, None], torch.zeros(1, 6, 1, device=DEV),
                                                       ops.rotary_tables(3, 64, device=DEV))),
        ("cos must be", lambda: ops.head_rotary_fwd(t[:, :, None], torch.zeros(1, 6, 2, device=DEV).long(),
                                                    ops.rotary_tables(3, 64, device=DEV))),
        ("rotary_dim", lambda: ops.head_rotary_fwd(t[:, :, None], torch.zeros(1, 6, 1, device=DEV).long(),
                                                   ops.rotary_tables(3, 64, device=DEV), rotary_dim=66)),
        ("weight must be", lambda: ops.head_rotary_fwd(t[:, :, None], norm=True, weight=torch.ones(64, device=DEV))),
        ("one dtype", lambda: ops.head_rotary_fwd(t[:, :, None], norm=True, weight=torch.ones(1, 64, device=DEV),
                                                  bias=torch.ones(1, 64, device=DEV).to(BF))),
        ("out must be", lambda: ops.head_rotary_bwd(t[:, :, None], t[:, :, None], norm=True, out=t)),
        ("dy must be", lambda: ops.head_rotary_bwd(t[:, :, None].float(), t[:, :, None], norm=True)),
        ("float32, bfloat16 or float16", lambda: ops.layer_norm_fwd(t.double())),
        ("rows give", lambda: ops.layer_norm_fwd(t, out_dtype=torch.float32)),
        ("weight must be", lambda: ops.layer_norm_fwd(t, torch.ones(63, device=DEV))),
        ("dy must be like", lambda: ops.layer_norm_bwd(t[:, :5], t, lse, lse)),
        ("mean must be", lambda: ops.layer_norm_bwd(t, t, lse, lse)),
    ]
    for match, call in bad:
        with pytest.raises(ValueError, match=match):
            call()
    for match, call in (("rows of", lambda: ops.layer_norm_fwd(torch.zeros(2, 8200, device=DEV))),
                        ("rows of", lambda: ops.head_rotary_fwd(torch.zeros(1, 1, 1, 1, 130, device=DEV), norm=True)),
                        ("pattern", lambda: ops.frame_attn_fwd(t, t, t, [0, ops.KEYSET]))):
        with pytest.raises(RuntimeError, match=match):
            call()
