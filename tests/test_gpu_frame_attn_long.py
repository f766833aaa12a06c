"""Attention over as many tokens as the aggregator's global layers have over 64 and 128 frames of 518 x 518, with
gradients: every row of one head against 64 bits."""
import importlib

import pytest
import torch

import train_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def ops(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return importlib.import_module(pkg.__name__ + ".ops")


def dense64(q, k, v, do, rows=4096):
    """Results of a dense head in 64 bits, a few query rows at a time."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    res = {n: torch.empty_like(q) for n in ("out", "dq")}
    res.update({n: torch.zeros_like(k) for n in ("dk", "dv")})
    res["lse"] = torch.empty(q.shape[0], dtype=torch.float64, device=q.device)
    kt, vt = k.t().contiguous(), v.t().contiguous()
    for at in range(0, q.shape[0], rows):
        sl = slice(at, at + rows)
        s = torch.mm(q[sl], kt).mul_(0.125)
        lse = torch.logsumexp(s, -1)
        p = s.sub_(lse[:, None]).exp_()
        out = torch.mm(p, v)
        ds = torch.mm(do[sl], vt).sub_((do[sl] * out).sum(-1, keepdim=True)).mul_(p).mul_(0.125)
        res["lse"][sl], res["out"][sl], res["dq"][sl] = lse, out, torch.mm(ds, k)
        res["dv"] += torch.mm(p.t().contiguous(), do[sl])
        res["dk"] += torch.mm(ds.t().contiguous(), q[sl])
    return res


@pytest.mark.parametrize("frames,masked", [(64, False), (64, True), (128, False)])
def test_global_layers_of_many_frames(ops, frames, masked):
    T, H = 1374, 2
    N = frames * T
    g = torch.Generator(device=DEV).manual_seed(frames)
    shared = torch.randn(1, T, H, 64, generator=g, device=DEV)
    q, k = (0.8 * shared.repeat(1, frames, 1, 1) + 0.6 * torch.randn(1, N, H, 64, generator=g, device=DEV) for _ in "qk")
    q, k, v, do = (t.to(BF) for t in (q, k, *(torch.randn(1, N, H, 64, generator=g, device=DEV) for _ in "vd")))
    mask = None
    there = torch.ones(N, dtype=torch.bool, device=DEV)
    if masked:  # frames of several heights, some views missing
        lengths = torch.tensor([0 if f % 9 == 4 else T - (f * 37 % 5) * T // 9 for f in range(frames)], device=DEV)
        there = (torch.arange(T, device=DEV) < lengths[:, None]).flatten()
        mask = there[None].clone()
        for t in (q, k, v, do):
            t[:, ~there] = float("nan")
    patterns = [ops.ANCHOR_LOCAL, ops.DENSE]
    out, lse, rest = ops.frame_attn_fwd(q, k, v, patterns, frames, mask, rest=True)
    dq, dk, dv = ops.frame_attn_bwd(do, q, k, v, out, lse, patterns, frames, mask, rest=rest)
    want = dense64(*(t[0, there, 1] for t in (q, k, v, do)))
    top = want["lse"].abs().max()
    # fp32 sums of N probabilities, and scores of 64 products
    assert (lse[0, 1, there] - want["lse"]).abs().max() < (N + 72) * R.E32 * top
    # parts of the rows by themselves, so that a wrong stretch is not lost in the whole
    n = want["out"].shape[0]
    parts = [slice(0, n), slice(0, 300), slice(n // 2, n // 2 + 300), slice(n - 300, n)]
    for name, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        assert not t[0, ~there].any(), name
        for sl in parts:
            w = want[name][sl]
            rel = float((t[0, there, 1][sl].double() - w).norm() / w.norm())
            # a result's rounding and its operands' (P, dS, D), each at most U of magnitudes that add in quadrature
            assert rel < 2 * R.U, (name, sl, rel)
