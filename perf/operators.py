"""Operators of a training step of the head-wise sparse attention layers, measured through the package's public entry
points, next to their plain forms in elementary torch operations.

Kinds
-----
attn      attention over the tokens of frames with a pattern per head (dense, frame-local, anchor + local, anchor),
          forward (output and log-sum-exp) or a training step (those and the gradients of q, k and v).
rotary    LayerNorm over the head dimension and rotary positions of q and k as they lie in a qkv buffer, forward or a
          training step (gradients of the rows and of the norm's parameters).
norm      LayerNorm over the model dimension, forward or a training step.

Clips of a batch may be padded: a token mask removes padded tokens, whose rows hold whatever the buffer held.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

HEAD_DIM = 64
NS = 5  # camera and register tokens of a frame
EPS = 1e-5
PATTERNS = ("dense", "local", "anchor_local", "anchor")  # also the keys of a case's head counts
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MAX_PAIRS = 16 * (12 * 1374) ** 2  # token pairs x heads of the largest attention case


def _ops():
    import __graft_entry__
    return importlib.import_module(__graft_entry__.package().__name__ + ".ops")


# ---- cases ----------------------------------------------------------------------------------------------

def listed():
    return [
        # two small views in one global layer: the smallest step, bound by launches and latency
        {"name": "attn_train_2x261", "kind": "attn", "train": True, "clips": 1, "frames": 2, "tokens": 261,
         "dense": 16, "local": 0, "anchor_local": 0, "anchor": 0, "pad": 0},
        # frame attention of eight 518 x 518 frames: every frame a sequence of its own
        {"name": "attn_train_frames_8x1374", "kind": "attn", "train": True, "clips": 8, "frames": 1, "tokens": 1374,
         "dense": 16, "local": 0, "anchor_local": 0, "anchor": 0, "pad": 0},
        # a global layer under a head profile, two clips of six 392 x 518 views, frames cropped to several sizes, one
        # clip with a missing first view
        {"name": "attn_train_mix_2x6x1041", "kind": "attn", "train": True, "clips": 2, "frames": 6, "tokens": 1041,
         "dense": 4, "local": 5, "anchor_local": 4, "anchor": 3, "pad": 3},
        # inference of a global layer with the statistics, 24 heads of the giant shape at 504 x 504
        {"name": "attn_fwd_8x1301", "kind": "attn", "train": False, "clips": 1, "frames": 8, "tokens": 1301,
         "dense": 12, "local": 6, "anchor_local": 6, "anchor": 0, "pad": 0},
        # a dense-heavy global layer over twelve 518 x 518 frames: the largest step
        {"name": "attn_train_12x1374", "kind": "attn", "train": True, "clips": 1, "frames": 12, "tokens": 1374,
         "dense": 10, "local": 2, "anchor_local": 2, "anchor": 2, "pad": 0},
        # q and k of one 392 x 518 view, forward: latency
        {"name": "rotary_fwd_1x1041", "kind": "rotary", "train": False, "clips": 1, "tokens": 1041, "groups": 2,
         "heads": 16, "dim": 64, "axes": 2, "rotary_dim": 64, "layout": "half", "norm": True, "dtype": "bf16"},
        # q and k of a global layer over sixteen 518 x 518 frames
        {"name": "rotary_train_16x1374", "kind": "rotary", "train": True, "clips": 16, "tokens": 1374, "groups": 2,
         "heads": 16, "dim": 64, "axes": 2, "rotary_dim": 64, "layout": "half", "norm": True, "dtype": "bf16"},
        # a temporal axis: far positions, interleaved pairs, half of a wider head, full precision
        {"name": "rotary_train_long_fp32", "kind": "rotary", "train": True, "clips": 3, "tokens": 4099, "groups": 2,
         "heads": 12, "dim": 128, "axes": 1, "rotary_dim": 64, "layout": "interleaved", "norm": False,
         "dtype": "fp32"},
        # a block's norm over one 392 x 518 view
        {"name": "norm_fwd_1041x1024", "kind": "norm", "train": False, "rows": 1041, "dim": 1024, "dtype": "bf16",
         "out": "bf16"},
        # a block's norm on an fp32 residual stream of 64 frames of 518 x 518, 16-bit output for the next product
        {"name": "norm_train_87936x1024", "kind": "norm", "train": True, "rows": 64 * 1374, "dim": 1024,
         "dtype": "fp32", "out": "bf16"},
        # the giant's width, half precision
        {"name": "norm_train_10408x1536_fp16", "kind": "norm", "train": True, "rows": 8 * 1301, "dim": 1536,
         "dtype": "fp16", "out": "fp16"},
        # a width that no vector divides
        {"name": "norm_train_4097x1027_fp32", "kind": "norm", "train": True, "rows": 4097, "dim": 1027,
         "dtype": "fp32", "out": "fp32"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("attn", "attn", "attn", "rotary", "rotary", "norm", "norm"))
    train = rng.random() < 0.7
    if kind == "attn":
        total = rng.choice((1, 3, 12, 16, 16, 24))
        cuts = sorted(rng.randint(0, total) for _ in range(3))
        tokens = _log_int(rng, 2, 1500)  # (a lone key has a gradient of zero, which nothing can be compared with)
        clips = rng.choice((1, 1, 2, 3, 7))
        most = math.sqrt(MAX_PAIRS / (total * clips)) / tokens
        frames = _log_int(rng, 1, max(1, min(64, int(most))))
        return {"kind": "attn", "train": train, "clips": clips, "frames": frames, "tokens": tokens,
                "dense": cuts[0], "local": cuts[1] - cuts[0], "anchor_local": cuts[2] - cuts[1],
                "anchor": total - cuts[2], "pad": rng.choice((0, 0, 1, 2, 3))}
    if kind == "rotary":
        dim = rng.choice((64, 64, 64, 32, 96, 128))
        axes = rng.choice((1, 2, 2))
        rotary_dim = rng.choice((dim, dim, dim // 2))
        heads = rng.choice((1, 3, 12, 16, 24))
        tokens = _log_int(rng, 1, 5000)
        clips = _log_int(rng, 1, max(1, min(16, (16 * 1374 * 2 * 16 * 64) // (2 * heads * dim * tokens))))
        return {"kind": "rotary", "train": train, "clips": clips, "tokens": tokens, "groups": rng.choice((1, 2, 2)),
                "heads": heads, "dim": dim, "axes": axes, "rotary_dim": rotary_dim,
                "layout": rng.choice(("half", "half", "interleaved")), "norm": rng.random() < 0.7,
                "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32"))}
    dim = _log_int(rng, 16, 4096)
    if rng.random() < 0.7:
        dim = -(-dim // 64) * 64
    rows = _log_int(rng, 1, (64 * 1374 * 1024) // dim)
    dtype, out = rng.choice((("bf16", "bf16"), ("fp32", "bf16"), ("fp32", "fp32"), ("fp16", "fp16"), ("fp32", "fp16")))
    return {"kind": "norm", "train": train, "rows": rows, "dim": dim, "dtype": dtype, "out": out}


def _heads(case):
    """Heads of every pattern."""
    return [case[p] for p in PATTERNS]


def _lengths(case):
    """Valid tokens of every frame of every clip, [clips][frames]; the rest of a frame's rows is padding."""
    T, res = case["tokens"], []
    for c in range(case["clips"]):
        row = []
        for f in range(case["frames"]):
            n = T
            if case["pad"] >= 1:  # frames of other aspect ratios
                n = max(1, T - ((f * 37 + c * 101) % 5) * T // 9)
            if case["pad"] >= 2 and case["frames"] > 2 and f == case["frames"] - 1 and c % 2 == 0:
                n = 0  # a shorter clip
            if case["pad"] >= 3 and c % 2 == 1 and f == 0:
                n = 0  # a clip whose first view is missing
            row.append(n)
        res.append(row)
    return res


def work(case):
    if case["kind"] == "attn":
        dense, local, anchor_local, anchor = _heads(case)
        pairs = 0
        for lens in _lengths(case):
            n, own_frame, first = sum(lens), sum(x * x for x in lens), lens[0]
            pairs += dense * n * n + local * own_frame + anchor * n * first
            pairs += anchor_local * (n * first + own_frame - first * first)
        rows = case["clips"] * case["frames"] * case["tokens"] * sum(_heads(case))
        tensors = 8 if case["train"] else 4
        products = 7 if case["train"] else 2
        return {"bytes": rows * (tensors * HEAD_DIM * 2.0 + 4), "flops": 2.0 * products * HEAD_DIM * pairs}
    if case["kind"] == "rotary":
        n = case["clips"] * case["tokens"]
        values = float(n * case["groups"] * case["heads"] * case["dim"])
        size = DTYPES[case["dtype"]].itemsize
        return {"bytes": values * size * (4 if case["train"] else 2) + n * case["axes"] * 8,
                "flops": values * (24 if case["train"] else 10)}
    values = float(case["rows"] * case["dim"])
    a, b = DTYPES[case["dtype"]].itemsize, DTYPES[case["out"]].itemsize
    return {"bytes": values * ((2 * a + 2 * b) if case["train"] else (a + b)) + case["rows"] * 8,
            "flops": values * (20 if case["train"] else 8)}


# ---- inputs ---------------------------------------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _tables(case):
    """cos / sin of position x inverse frequency, from 64-bit angles. Patch grids: base 100, as the model's 2-D
    positions; the temporal axis: base 10000 with positions up to 2^20, scaled to four times the trained range."""
    S = case["rotary_dim"] // case["axes"]
    n = 64 if case["axes"] == 2 else 1 << 16
    base = 100.0 if case["axes"] == 2 else 10000.0
    scale = 1.0 if case["axes"] == 2 else 0.25
    j = torch.arange(0, S, 2, dtype=torch.float64, device="cuda")
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * scale / base ** (j / S)
    return ang.cos().float(), ang.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "attn":
        B, F, T, H = case["clips"], case["frames"], case["tokens"], sum(_heads(case))
        N = F * T
        # normed and rotated q and k: content shared by the frames, so that a token has near matches in every view
        shared = _randn(g, B, 1, T, 1, H, HEAD_DIM)
        qk = 0.8 * shared + 0.6 * _randn(g, B, F, T, 2, H, HEAD_DIM)
        qk = qk.reshape(B, N, 2, H, HEAD_DIM).to(torch.bfloat16)
        qkv = (_randn(g, B, N, 3, H, HEAD_DIM) + 0.3 * _randn(g, 1, 1, 3, H, HEAD_DIM)).to(torch.bfloat16)
        dout = (0.01 * _randn(g, B, N, H, HEAD_DIM)).to(torch.bfloat16)
        mask = None
        if case["pad"]:
            lens = torch.tensor(_lengths(case), device="cuda")
            mask = (torch.arange(T, device="cuda") < lens[..., None]).reshape(B, N)
            qk[~mask] = math.nan
            qkv[~mask] = math.inf
            dout[~mask] = 0
        order = [p for p, n in enumerate(_heads(case)) for _ in range(n)]
        perm = torch.randperm(H, generator=g, device="cuda").tolist()
        return {"case": case, "q": qk[:, :, 0], "k": qk[:, :, 1], "v": qkv[:, :, 2], "dout": dout, "mask": mask,
                "patterns": [order[i] for i in perm], "pattern_ids": torch.tensor(order, device="cuda")[perm]}
    if kind == "rotary":
        B, N, G, H, D = case["clips"], case["tokens"], case["groups"], case["heads"], case["dim"]
        dt = DTYPES[case["dtype"]]
        qkv = (1.5 * _randn(g, B, N, 3, H, D) + 0.5 * _randn(g, 1, 1, 3, H, D)).to(dt)
        if case["axes"] == 2:  # (row + 1, column + 1) of a patch grid, the camera and register tokens at 0
            w = 37
            p = (torch.arange(N, device="cuda") - NS).clamp(min=-1)
            pos = torch.stack([torch.where(p < 0, 0, p // w % 60 + 1), torch.where(p < 0, 0, p % w + 1)], dim=-1)
            pos = pos.expand(B, N, 2).contiguous()
        else:
            start = torch.randint(0, (1 << 16) - N, (B, 1), generator=g, device="cuda")
            pos = (start + torch.arange(N, device="cuda"))[..., None].contiguous()
        cos, sin = _tables(case)
        state = {"case": case, "x": qkv[:, :, :G], "pos": pos, "cos": cos, "sin": sin, "weight": None, "bias": None,
                 "dy": (0.01 * _randn(g, B, N, G, H, D)).to(dt)}
        if case["norm"]:
            state["weight"] = 1 + 0.2 * _randn(g, G, D)
            state["bias"] = 0.1 * _randn(g, G, D)
        return state
    R, C = case["rows"], case["dim"]
    # a residual stream: tokens of several magnitudes and offsets, a few large channels
    x = _randn(g, R, C) * (0.5 + torch.rand(R, 1, generator=g, device="cuda") * 4) + _randn(g, R, 1)
    x[:, torch.randint(0, C, (max(1, C // 256),), generator=g, device="cuda")] *= 8
    return {"case": case, "x": x.to(DTYPES[case["dtype"]]), "weight": 1 + 0.2 * _randn(g, C),
            "bias": 0.1 * _randn(g, C), "dy": (0.01 * _randn(g, R, C)).to(DTYPES[case["out"]])}


# ---- one pass -------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return {"attn": _own_attn, "rotary": _own_rotary, "norm": _own_norm}[case["kind"]](state)
    return {"attn": _plain_attn, "rotary": _plain_rotary, "norm": _plain_norm}[case["kind"]](state)


def _own_attn(s):
    ops, case = _ops(), s["case"]
    ids = (ops.DENSE, ops.FRAME_LOCAL, ops.ANCHOR_LOCAL, ops.ANCHOR)
    patterns = [ids[p] for p in s["patterns"]]
    args = dict(frames=case["frames"], token_mask=s["mask"])
    if not case["train"]:
        out, lse = ops.frame_attn_fwd(s["q"], s["k"], s["v"], patterns, **args)
        return {"out": out, "lse": lse}
    out, lse, rest = ops.frame_attn_fwd(s["q"], s["k"], s["v"], patterns, rest=True, **args)
    dq, dk, dv = ops.frame_attn_bwd(s["dout"], s["q"], s["k"], s["v"], out, lse, patterns, rest=rest, **args)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _own_rotary(s):
    ops, case = _ops(), s["case"]
    args = dict(pos=s["pos"], tables=(s["cos"], s["sin"]), layout=case["layout"], rotary_dim=case["rotary_dim"],
                norm=case["norm"], weight=s["weight"], eps=EPS)
    y = ops.head_rotary_fwd(s["x"], bias=s["bias"], **args)
    if not case["train"]:
        return {"y": y}
    dx, dweight, dbias = ops.head_rotary_bwd(s["dy"], s["x"], **args)
    return {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias} if case["norm"] else {"y": y, "dx": dx}


def _own_norm(s):
    ops, case = _ops(), s["case"]
    y, mean, rstd = ops.layer_norm_fwd(s["x"], s["weight"], s["bias"], eps=EPS, out_dtype=DTYPES[case["out"]])
    if not case["train"]:
        return {"y": y}
    dx, dweight, dbias = ops.layer_norm_bwd(s["dy"], s["x"], mean, rstd, s["weight"])
    return {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias}


def _allowed(case, pattern_ids, mask):
    """[B or 1, H, N, N]: whether query i of a head may attend key j."""
    frame = torch.arange(case["frames"] * case["tokens"], device="cuda") // case["tokens"]
    same, first = frame[:, None] == frame[None, :], (frame == 0)[None, :]
    pid = pattern_ids[:, None, None]
    ok = (pid == 0) | (same & ((pid == 1) | (pid == 2))) | (first & ((pid == 2) | (pid == 3)))
    ok = ok[None]
    return ok if mask is None else ok & (mask[:, None, :, None] & mask[:, None, None, :])


def _plain_attn(s):
    case, mask = s["case"], s["mask"]
    q, k, v, do = (t.float().transpose(1, 2) for t in (s["q"], s["k"], s["v"], s["dout"]))  # [B, H, N, 64]
    if mask is not None:
        keep = mask[:, None, :, None]
        q, k, v, do = (torch.where(keep, t, 0.0) for t in (q, k, v, do))
    q, k, v, do = (t.contiguous() for t in (q, k, v, do))
    scale = HEAD_DIM ** -0.5
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    p.masked_fill_(~_allowed(case, s["pattern_ids"], mask), -math.inf)
    m = p.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    lse = (m + torch.log(l)).squeeze(-1)
    p.mul_(torch.where(l > 0, 1.0 / l, 0.0))
    o = torch.matmul(p, v)
    out = o.transpose(1, 2).to(torch.bfloat16)
    if not case["train"]:
        return {"out": out, "lse": lse}
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    del p
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3), q)
    return {"out": out, "lse": lse, **{n: t.transpose(1, 2).to(torch.bfloat16)
                                       for n, t in (("dq", dq), ("dk", dk), ("dv", dv))}}


def _angles(s, sign=1.0):
    """cos and sin of every rotated pair, [B, N, 1, 1, axes, S / 2]."""
    return s["cos"][s["pos"]][:, :, None, None], sign * s["sin"][s["pos"]][:, :, None, None]


def _rotate(case, x, cos, sin):
    R, A = case["rotary_dim"], case["axes"]
    part = x[..., :R].unflatten(-1, (A, R // A))
    if case["layout"] == "half":
        a, b = part.chunk(2, dim=-1)
        part = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([part.flatten(-2), x[..., R:]], dim=-1)


def _plain_rotary(s):
    case, x = s["case"], s["x"].float()
    y = x
    if case["norm"]:
        c = x - x.mean(-1, keepdim=True)
        r = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
        xh = c * r
        w = s["weight"][:, None]
        y = xh * w + s["bias"][:, None]
    y = _rotate(case, y, *_angles(s)).to(s["x"].dtype)
    if not case["train"]:
        return {"y": y}
    dy = _rotate(case, s["dy"].float(), *_angles(s, -1.0))  # the inverse rotation
    if not case["norm"]:
        return {"y": y, "dx": dy.to(s["x"].dtype)}
    gx = dy * w
    dx = r * (gx - gx.mean(-1, keepdim=True) - xh * (gx * xh).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dweight": (dy * xh).sum((0, 1, 3)), "dbias": dy.sum((0, 1, 3))}


def _plain_norm(s):
    case, x, w = s["case"], s["x"].float(), s["weight"]
    c = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    xh = c * r
    y = (xh * w + s["bias"]).to(DTYPES[case["out"]])
    if not case["train"]:
        return {"y": y}
    dy = s["dy"].float()
    gx = dy * w
    dx = r * (gx - gx.mean(-1, keepdim=True) - xh * (gx * xh).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dweight": (dy * xh).sum(0), "dbias": dy.sum(0)}


# ---- the same in 64 bits --------------------------------------------------------------------------------

def _exact_attn(s):
    """One head of one clip at a time, over the tokens that are there and the keys that a frame's queries see."""
    case = s["case"]
    B, F, T, H = case["clips"], case["frames"], case["tokens"], sum(_heads(case))
    N = F * T
    shape = (B, N, H, HEAD_DIM)
    res = {n: torch.zeros(shape, dtype=torch.float64, device="cuda") for n in ("out", "dq", "dk", "dv")}
    lse = torch.full((B, H, N), -math.inf, dtype=torch.float64, device="cuda")
    everything = torch.arange(N, device="cuda")
    for b, lens in enumerate(_lengths(case)):
        frames = [everything[f * T:f * T + n] for f, n in enumerate(lens)]
        there = torch.cat(frames)
        for h, p in enumerate(s["patterns"]):
            name = PATTERNS[p]
            if name == "dense":
                jobs = [(part, there) for part in there.split(8192)]
            elif name == "anchor":
                jobs = [(there, frames[0])]
            else:
                seen = [f if name == "local" or i == 0 else torch.cat([frames[0], f]) for i, f in enumerate(frames)]
                jobs = list(zip(frames, seen))
            for rows, keys in jobs:
                if rows.numel() == 0 or keys.numel() == 0:
                    continue
                q, do = s["q"][b, rows, h].double(), s["dout"][b, rows, h].double()
                k, v = s["k"][b, keys, h].double(), s["v"][b, keys, h].double()
                x = torch.mm(q, k.t().contiguous()) / math.sqrt(HEAD_DIM)
                lse[b, h, rows] = torch.logsumexp(x, dim=-1)
                pr = torch.softmax(x, dim=-1)
                o = torch.mm(pr, v)
                res["out"][b, rows, h] = o
                if case["train"]:
                    dx = pr * (torch.mm(do, v.t().contiguous()) - (do * o).sum(-1, keepdim=True)) / math.sqrt(HEAD_DIM)
                    res["dq"][b, rows, h] = torch.mm(dx, k)
                    res["dk"][b, keys, h] += torch.mm(dx.t().contiguous(), q)
                    res["dv"][b, keys, h] += torch.mm(pr.t().contiguous(), do)
    if not case["train"]:
        return {"out": res["out"], "lse": lse}
    return {"out": res["out"], "lse": lse, "dq": res["dq"], "dk": res["dk"], "dv": res["dv"]}


def _layer_norm64(x, weight, bias):
    return torch.nn.functional.layer_norm(x, x.shape[-1:], None, None, EPS) * weight + bias


def _exact_rotary(s):
    """Pairs as complex numbers; the gradients by torch's differentiation in 64 bits."""
    case = s["case"]
    R, A = case["rotary_dim"], case["axes"]
    S = R // A
    turn = torch.complex(s["cos"].double()[s["pos"]], s["sin"].double()[s["pos"]])[:, :, None, None]
    x = s["x"].double().requires_grad_(case["train"])
    leaves = [x]
    y = x
    if case["norm"]:
        w, bias = (s[n].double().requires_grad_(case["train"]) for n in ("weight", "bias"))
        leaves += [w, bias]
        y = _layer_norm64(x, w[:, None], bias[:, None])
    z = y[..., :R].reshape(*y.shape[:-1], A, S)
    z = z.unflatten(-1, (2, S // 2)).transpose(-1, -2) if case["layout"] == "half" else z.unflatten(-1, (S // 2, 2))
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
    z = z.transpose(-1, -2) if case["layout"] == "half" else z
    y = torch.cat([z.reshape(*y.shape[:-1], R), y[..., R:]], dim=-1)
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, leaves, s["dy"].double())
    return dict(zip(("y", "dx", "dweight", "dbias"), (y.detach(), *grads)))


def _exact_norm(s):
    case = s["case"]
    x, w, bias = (s[n].double().requires_grad_(case["train"]) for n in ("x", "weight", "bias"))
    y = _layer_norm64(x, w, bias)
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, (x, w, bias), s["dy"].double())
    return dict(zip(("y", "dx", "dweight", "dbias"), (y.detach(), *grads)))


def exact(case, seed):
    state = prepare(case, seed)
    return {"attn": _exact_attn, "rotary": _exact_rotary, "norm": _exact_norm}[case["kind"]](state)
