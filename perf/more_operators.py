"""Operators of a transformer block around its attention, measured through the package's public entry points, next to
their plain forms in elementary torch operations.

Kinds
-----
linear    product with a weight, and in its epilogue bias, activation, dropout, gate (a layer scale) and residual:
          y = residual + gate drop(act(x W^T + bias)), forward or a training step (gradients of x, the weight, the bias
          and the gate; the residual's is dy itself).
residual  gated residual and the norm of the rows that come out: h = x + gate drop(branch), y = LayerNorm(h), forward or a
          training step (gradients of x, the branch, the gate and the norm's parameters). h is rounded to the stream's
          type before the norm, which normalises the stream as the next block will read it.
dropout   y = x keep / (1 - p), forward or a training step.

The keep mask is a function of (state, row, column): sixteen bits of Philox4x32-10 (Salmon et al., 2011) for every element,
compared with round(65536 p); the state (seed, stream) is an input.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_PRODUCTS = 3 * 64 * 1374 * 1024 * 4096  # of the largest linear case
MOST_VALUES = 64 * 1374 * 1024  # of the largest case of the other kinds


def _ops():
    import __graft_entry__
    return importlib.import_module(__graft_entry__.package().__name__ + ".ops")


# ---- cases ----------------------------------------------------------------------------------------------

def listed():
    return [
        # the first MLP product on the camera tokens of four views: latency
        {"name": "linear_fwd_4x1024x4096", "kind": "linear", "train": False, "rows": 4, "in": 1024, "out": 4096,
         "act": "gelu", "gate": False, "residual": "", "p": 0.0, "dtype": "bf16"},
        # the attention's output product into an fp32 residual stream, two small views
        {"name": "linear_fwd_522x1024x1024", "kind": "linear", "train": False, "rows": 522, "in": 1024, "out": 1024,
         "act": "", "gate": True, "residual": "fp32", "p": 0.0, "dtype": "bf16"},
        # the first MLP product of one 392 x 518 view, a training step
        {"name": "linear_train_1041x1024x4096", "kind": "linear", "train": True, "rows": 1041, "in": 1024, "out": 4096,
         "act": "gelu", "gate": False, "residual": "", "p": 0.0, "dtype": "bf16"},
        # the second one over eight 518 x 518 frames with dropout, layer scale and residual
        {"name": "linear_train_10992x4096x1024", "kind": "linear", "train": True, "rows": 8 * 1374, "in": 4096,
         "out": 1024, "act": "", "gate": True, "residual": "fp32", "p": 0.1, "dtype": "bf16"},
        # the giant's width at inference, 504 x 504, half precision
        {"name": "linear_fwd_10408x1536x6144_fp16", "kind": "linear", "train": False, "rows": 8 * 1301, "in": 1536,
         "out": 6144, "act": "gelu", "gate": False, "residual": "", "p": 0.0, "dtype": "fp16"},
        # widths that no tile or vector divides
        {"name": "linear_train_777x1027x515", "kind": "linear", "train": True, "rows": 777, "in": 1027, "out": 515,
         "act": "gelu_tanh", "gate": True, "residual": "bf16", "p": 0.0, "dtype": "bf16"},
        # the first MLP product over 64 frames of 518 x 518: the largest step
        {"name": "linear_train_87936x1024x4096", "kind": "linear", "train": True, "rows": 64 * 1374, "in": 1024,
         "out": 4096, "act": "gelu", "gate": False, "residual": "", "p": 0.0, "dtype": "bf16"},
        # between attention and MLP of one 392 x 518 view: latency
        {"name": "residual_fwd_1041x1024", "kind": "residual", "train": False, "rows": 1041, "dim": 1024, "gate": True,
         "p": 0.0, "dtype": "bf16", "out": "bf16"},
        # the same in a training step on an fp32 residual stream of 64 frames of 518 x 518
        {"name": "residual_train_87936x1024", "kind": "residual", "train": True, "rows": 64 * 1374, "dim": 1024,
         "gate": True, "p": 0.0, "dtype": "fp32", "out": "bf16"},
        # the giant's width, half precision, dropout
        {"name": "residual_train_10408x1536_fp16", "kind": "residual", "train": True, "rows": 8 * 1301, "dim": 1536,
         "gate": True, "p": 0.1, "dtype": "fp16", "out": "fp16"},
        # dropout of one 392 x 518 view's tokens: latency
        {"name": "dropout_fwd_1041x1024", "kind": "dropout", "train": False, "rows": 1041, "dim": 1024, "p": 0.1,
         "dtype": "bf16"},
        # and of 64 frames of 518 x 518 in a training step
        {"name": "dropout_train_87936x1024", "kind": "dropout", "train": True, "rows": 64 * 1374, "dim": 1024,
         "p": 0.25, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    n = _log_int(rng, lo, hi)
    return -(-n // 64) * 64 if rng.random() < 0.7 else n


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear", "residual", "residual", "dropout"))
    train = rng.random() < 0.6
    p = rng.choice((0.0, 0.0, 0.05, 0.1, 0.3))
    if kind == "linear":
        k, n = _width(rng, 32, 6144), _width(rng, 32, 6144)
        rows = _log_int(rng, 1, max(1, min(64 * 1374, MOST_PRODUCTS // ((3 if train else 1) * k * n))))
        dtype = rng.choice(("bf16", "bf16", "fp16"))
        residual = rng.choice(("", "fp32", dtype))
        return {"kind": kind, "train": train, "rows": rows, "in": k, "out": n,
                "act": rng.choice(("", "gelu", "gelu", "gelu_tanh")), "gate": rng.random() < 0.5, "residual": residual,
                "p": p, "dtype": dtype}
    dim = _width(rng, 16, 4096)
    rows = _log_int(rng, 1, MOST_VALUES // dim)
    if kind == "dropout":
        return {"kind": kind, "train": train, "rows": rows, "dim": dim, "p": rng.choice((0.05, 0.1, 0.25, 0.5)),
                "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32"))}
    dtype, out = rng.choice((("bf16", "bf16"), ("fp32", "bf16"), ("fp32", "fp32"), ("fp16", "fp16"), ("fp32", "fp16")))
    return {"kind": kind, "train": train, "rows": rows, "dim": dim, "gate": rng.random() < 0.8, "p": p, "dtype": dtype,
            "out": out}


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "linear":
        R, K, N = float(case["rows"]), case["in"], case["out"]
        res = DTYPES[case["residual"]].itemsize if case["residual"] else 0
        moved = size * (R * K + N * K) + R * N * (2 * res if res else size)
        if case["train"]:  # dy is read; dx and dW are written
            moved += R * N * (res or size) + size * (R * K + N * K)
        return {"bytes": moved, "flops": 2 * R * K * N * (3 if case["train"] else 1)}
    values = float(case["rows"] * case["dim"])
    if case["kind"] == "dropout":
        return {"bytes": values * size * (4 if case["train"] else 2), "flops": values * (2 if case["train"] else 1)}
    out = DTYPES[case["out"]].itemsize
    # x and the branch, h and y; then dh and dy, dx and dbranch
    return {"bytes": values * (2 * size + 2 * out) * (2 if case["train"] else 1),
            "flops": values * (34 if case["train"] else 10)}


# ---- inputs ---------------------------------------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, dt, R = case["kind"], DTYPES[case["dtype"]], case["rows"]
    state = torch.randint(0, 1 << 62, (2,), generator=g, device="cuda")
    if kind == "linear":
        K, N = case["in"], case["out"]
        s = {"case": case, "state": state, "gate": None, "residual": None}
        s["x"] = (_randn(g, R, K) * (1 + 0.2 * _randn(g, K)) + 0.1 * _randn(g, K)).to(dt)  # rows of a norm
        s["weight"] = (_randn(g, N, K) / math.sqrt(K)).to(dt)
        s["bias"] = (0.2 * _randn(g, N)).to(dt)
        if case["gate"]:
            s["gate"] = (0.1 + 0.4 * torch.rand(N, generator=g, device="cuda")).to(dt)
        out = dt
        if case["residual"]:
            out = DTYPES[case["residual"]]
            s["residual"] = (2 * _randn(g, R, N)).to(out)
        s["dy"] = (0.01 * _randn(g, R, N) + 0.002 * _randn(g, N)).to(out)
        return s
    C = case["dim"]
    if kind == "dropout":
        return {"case": case, "state": state, "x": _randn(g, R, C).to(dt), "dy": (0.01 * _randn(g, R, C)).to(dt)}
    out = DTYPES[case["out"]]
    # a residual stream: tokens of several magnitudes and offsets; a branch in the type of the products
    x = _randn(g, R, C) * (0.5 + torch.rand(R, 1, generator=g, device="cuda") * 4) + _randn(g, R, 1)
    return {"case": case, "state": state, "x": x.to(dt), "branch": _randn(g, R, C).to(out),
            "gate": (0.1 + 0.4 * torch.rand(C, generator=g, device="cuda")).to(dt) if case["gate"] else None,
            "weight": (1 + 0.2 * _randn(g, C)).to(dt), "bias": (0.1 * _randn(g, C)).to(dt),
            "dh": (0.01 * _randn(g, R, C) + 0.002 * _randn(g, C)).to(dt), "dy": (0.01 * _randn(g, R, C)).to(out)}


# ---- one pass -------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return {"linear": _own_linear, "residual": _own_residual, "dropout": _own_dropout}[case["kind"]](state)
    return {"linear": _plain_linear, "residual": _plain_residual, "dropout": _plain_dropout}[case["kind"]](state)


def _own_linear(s):
    ops, case = _ops(), s["case"]
    args = dict(activation=case["act"] or None, gate=s["gate"], dropout=case["p"], state=s["state"])
    if not case["train"]:
        return {"y": ops.linear_fwd(s["x"], s["weight"], s["bias"], residual=s["residual"], **args)}
    y, kept = ops.linear_fwd(s["x"], s["weight"], s["bias"], residual=s["residual"], keep=True, **args)
    dx, dweight, dbias, dgate = ops.linear_bwd(s["dy"], s["x"], s["weight"], kept, **args)
    grads = {"dx": dx, "dweight": dweight, "dbias": dbias}
    return {"y": y, **grads, "dgate": dgate} if case["gate"] else {"y": y, **grads}


def _own_residual(s):
    ops, case = _ops(), s["case"]
    args = dict(dropout=case["p"], state=s["state"])
    h, y, mean, rstd = ops.residual_norm_fwd(s["x"], s["branch"], s["gate"], s["weight"], s["bias"], eps=EPS,
                                             out_dtype=DTYPES[case["out"]], **args)
    if not case["train"]:
        return {"h": h, "y": y}
    dx, dbranch, dgate, dweight, dbias = ops.residual_norm_bwd(s["dh"], s["dy"], h, mean, rstd, s["branch"], s["gate"],
                                                               s["weight"], **args)
    grads = {"dx": dx, "dbranch": dbranch, "dweight": dweight, "dbias": dbias}
    return {"h": h, "y": y, **grads, "dgate": dgate} if case["gate"] else {"h": h, "y": y, **grads}


def _own_dropout(s):
    ops, case = _ops(), s["case"]
    y = ops.dropout(s["x"], case["p"], s["state"])
    return {"y": y, "dx": ops.dropout(s["dy"], case["p"], s["state"])} if case["train"] else {"y": y}


# ---- the plain forms ------------------------------------------------------------------------------------

M32 = 0xFFFFFFFF


def _philox(state, rows, cols):
    """Sixteen random bits for each of rows x cols elements (int64): word j / 2 of the block of counter
    (column / 8, row's low half, row's high half, stream), its low half for even j = column % 8."""
    seed, stream = state[0], state[1]
    groups = (cols + 7) // 8
    row = torch.arange(rows, device="cuda")[:, None]
    c0 = torch.arange(groups, device="cuda")[None, :].expand(rows, groups)
    c1, c2 = (row & M32).expand(rows, groups), (row >> 32).expand(rows, groups)
    c3 = (stream & M32).expand(rows, groups)
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # (their 64 bits, whatever the sign)
        c0, c1, c2, c3 = ((b >> 32) & M32) ^ c1 ^ k0, b & M32, ((a >> 32) & M32) ^ c3 ^ k1, a & M32
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    words = torch.stack([c0, c1, c2, c3], dim=-1)
    return torch.stack([words & 0xFFFF, words >> 16], dim=-1).reshape(rows, groups * 8)[:, :cols]


def _keep(s, cols, dtype=torch.float32):
    """keep / (1 - p) of every element, or 1 without dropout."""
    limit = round(s["case"]["p"] * 65536)
    if limit == 0:
        return 1.0
    return (_philox(s["state"], s["case"]["rows"], cols) >= limit).to(dtype) * (65536.0 / (65536 - limit))


def _plain_act(kind, z):
    """The activation and its derivative."""
    if kind == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return z, 1.0


def _plain_linear(s):
    case = s["case"]
    x, w = s["x"].float(), s["weight"].float()
    gate = 1.0 if s["gate"] is None else s["gate"].float()
    z = torch.matmul(x, w.t()) + s["bias"].float()
    a, slope = _plain_act(case["act"], z)
    keep = _keep(s, case["out"])
    a = a * keep
    y = gate * a
    if s["residual"] is not None:
        y = s["residual"].float() + y
    y = y.to(s["dy"].dtype)
    if not case["train"]:
        return {"y": y}
    dy, dt = s["dy"].float(), s["x"].dtype
    dz = dy * gate * keep * slope
    res = {"y": y, "dx": torch.matmul(dz, w).to(dt), "dweight": torch.matmul(dz.t(), x).to(dt), "dbias": dz.sum(0).to(dt)}
    if s["gate"] is not None:
        res["dgate"] = (dy * a).sum(0).to(dt)
    return res


def _plain_residual(s):
    case, dt, out = s["case"], s["x"].dtype, DTYPES[s["case"]["out"]]
    gate = 1.0 if s["gate"] is None else s["gate"].float()
    keep = _keep(s, case["dim"])
    b = s["branch"].float() * keep
    stream = (s["x"].float() + gate * b).to(dt)
    h, w = stream.float(), s["weight"].float()
    c = h - h.mean(-1, keepdim=True)
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    xh = c * r
    y = (xh * w + s["bias"].float()).to(out)
    if not case["train"]:
        return {"h": stream, "y": y}
    dy = s["dy"].float()
    gx = dy * w
    dh = s["dh"].float() + r * (gx - gx.mean(-1, keepdim=True) - xh * (gx * xh).mean(-1, keepdim=True))
    res = {"h": stream, "y": y, "dx": dh.to(dt), "dbranch": (gate * keep * dh).to(out),
           "dweight": (dy * xh).sum(0).to(dt), "dbias": dy.sum(0).to(dt)}
    if s["gate"] is not None:
        res["dgate"] = (dh * b).sum(0).to(dt)
    return res


def _plain_dropout(s):
    keep, dt = _keep(s, s["case"]["dim"]), s["x"].dtype
    y = (s["x"].float() * keep).to(dt)
    return {"y": y, "dx": (s["dy"].float() * keep).to(dt)} if s["case"]["train"] else {"y": y}


# ---- the same in 64 bits --------------------------------------------------------------------------------

def _mul32(a, m):
    """High and low words of a * m for words a in float64, by halves of sixteen bits (every step is exact)."""
    ah, al = torch.div(a, 65536, rounding_mode="floor"), torch.remainder(a, 65536)
    mh, ml = float(m >> 16), float(m & 0xFFFF)
    mid = ah * ml + al * mh + torch.div(al * ml, 65536, rounding_mode="floor")
    low = torch.remainder(al * ml, 65536) + torch.remainder(mid, 65536) * 65536
    return ah * mh + torch.div(mid, 65536, rounding_mode="floor"), low


def _exact_keep(s, cols):
    """The factor of every element; the generator on words held as float64, some rows at a time."""
    limit = round(s["case"]["p"] * 65536)
    if limit == 0:
        return torch.ones((), dtype=torch.float64, device="cuda")
    seed, stream = (int(v) for v in s["state"].tolist())
    groups, parts = -(-cols // 8), []
    for rows in torch.arange(s["case"]["rows"], device="cuda").split(max(1, (1 << 22) // groups)):
        shape = (rows.numel(), groups)
        word = [torch.arange(groups, device="cuda", dtype=torch.float64).expand(shape),
                rows.to(torch.float64)[:, None].expand(shape),  # (fewer than 2^32 rows)
                torch.zeros(shape, dtype=torch.float64, device="cuda"),
                torch.full(shape, float(stream % 2 ** 32), dtype=torch.float64, device="cuda")]
        word = [w.contiguous() for w in word]
        for i in range(10):
            key = [((seed >> 32 * j) + i * w) % 2 ** 32 for j, w in enumerate((0x9E3779B9, 0xBB67AE85))]
            (ah, al), (bh, bl) = _mul32(word[0], 0xD2511F53), _mul32(word[2], 0xCD9E8D57)
            word = [(bh.long() ^ word[1].long() ^ key[0]).double(), bl,
                    (ah.long() ^ word[3].long() ^ key[1]).double(), al]
        bits = torch.empty(*shape, 8, dtype=torch.float64, device="cuda")
        for j in range(8):
            w = word[j // 2]
            bits[..., j] = torch.div(w, 65536, rounding_mode="floor") if j % 2 else torch.remainder(w, 65536)
        parts.append(bits.flatten(1)[:, :cols] >= limit)
    return torch.cat(parts).double() * (65536 / (65536 - limit))


def _given(s, *names):
    """Those inputs in 64 bits, asked for gradients in a training step."""
    return [None if s[n] is None else s[n].double().requires_grad_(s["case"]["train"]) for n in names]


def _results(s, outputs, upstream, names, leaves):
    """Outputs and, in a training step, the gradients by torch's differentiation."""
    if not s["case"]["train"]:
        return outputs
    there = [(n, t) for n, t in zip(names, leaves) if t is not None]
    grads = torch.autograd.grad(list(upstream), [t for _, t in there], list(upstream.values()))
    return {**{n: t.detach() for n, t in outputs.items()}, **dict(zip([n for n, _ in there], grads))}


def _exact_linear(s):
    case = s["case"]
    x, w, bias, gate = leaves = _given(s, "x", "weight", "bias", "gate")
    a = torch.nn.functional.linear(x, w, bias)
    if case["act"]:
        a = torch.nn.functional.gelu(a, approximate="tanh" if case["act"] == "gelu_tanh" else "none")
    y = a * _exact_keep(s, case["out"])
    y = y if gate is None else y * gate
    y = y if s["residual"] is None else y + s["residual"].double()
    return _results(s, {"y": y}, {y: s["dy"].double()}, ("dx", "dweight", "dbias", "dgate"), leaves)


def _exact_residual(s):
    branch, gate, w, bias = leaves = _given(s, "branch", "gate", "weight", "bias")
    b = branch * _exact_keep(s, s["case"]["dim"])
    h = s["x"].double() + (b if gate is None else b * gate)
    # the norm reads the stream as it is stored; its gradient passes the rounding
    stored = h.detach().to(s["x"].dtype).double()
    stored = stored + (h - h.detach())
    y = torch.nn.functional.layer_norm(stored, stored.shape[-1:], w, bias, EPS)
    # (the gradient of x is the one of h)
    return _results(s, {"h": h, "y": y}, {h: s["dh"].double(), y: s["dy"].double()},
                    ("dbranch", "dgate", "dweight", "dbias", "dx"), [*leaves, h])


def _exact_dropout(s):
    keep = _exact_keep(s, s["case"]["dim"])
    y = s["x"].double() * keep
    return {"y": y, "dx": s["dy"].double() * keep} if s["case"]["train"] else {"y": y}


def exact(case, seed):
    state = prepare(case, seed)
    return {"linear": _exact_linear, "residual": _exact_residual, "dropout": _exact_dropout}[case["kind"]](state)
