"""Calls of the block's operators (linear layers, gated residual with norm, dropout) that are refused, with the reason, before
anything is launched (CPU: the C entries with addresses that are never read; the wrappers' checks)."""
import ctypes
from importlib import import_module

import pytest
import torch

FP32, BF16, FP16 = 0, 1, 2
INVALID, UNSUPPORTED = 1, 2


@pytest.fixture(scope="module")
def L(pkg):
    return import_module(pkg.__name__ + "._lib")


def refused(L, rc, code, text):
    msg = L.load().saf3r_last_error().decode()
    assert rc == code and text in msg, (rc, msg)


def linear(L, bwd=False, x=256, xs=64, w=256, ws_=64, type=BF16, rows=3, k=64, n=32, bias=256, gate=256, pt=FP32, act=1,
           drop=100, state=256, res=256, rs=32, y=256, ys=32, yt=FP32, kept=256, ks=32, dy=256, dys=32, dx=256, dxs=64,
           dw=256, dws=64, dwt=FP32, db=256, dg=256, wsp=256, nbytes=1 << 20):
    lib = L.load()
    if bwd:
        return lib.saf3r_linear_bwd(dy, dys, yt, x, xs, w, ws_, type, rows, k, n, kept, ks, gate, pt, act, drop, state, dx,
                                    dxs, dw, dws, dwt, db, dg, wsp, nbytes, None)
    return lib.saf3r_linear_fwd(x, xs, w, ws_, type, rows, k, n, bias, gate, pt, act, drop, state, res, rs, y, ys, yt, kept,
                                ks, wsp, nbytes, None)


@pytest.mark.parametrize("bwd", [False, True])
def test_linear(L, bwd):
    def no(code, text, **kw):
        refused(L, linear(L, bwd, **kw), code, text)
    for kw in ({"rows": -1}, {"k": 0}, {"n": 0}, {"k": -8}):
        no(INVALID, "sizes", **kw)
    for kw in ({"k": (1 << 21) + 1}, {"n": (1 << 21) + 1}):
        no(UNSUPPORTED, "widths", **kw)
    no(UNSUPPORTED, "too many rows", rows=1 << 31)
    no(UNSUPPORTED, "bf16 or fp16", type=FP32)
    no(INVALID, "element type", type=3)
    no(INVALID, "element type", pt=7)
    no(INVALID, "element type", yt=-1)
    no(UNSUPPORTED, "fp32 or the operands' type", yt=FP16)
    no(UNSUPPORTED, "16-bit type", pt=FP16)
    no(INVALID, "activation", act=3)
    no(INVALID, "activation", act=-1)
    for drop in (-1, 65537):
        no(INVALID, "65536 times", drop=drop)
    no(INVALID, "state", state=None)
    no(INVALID, "state", state=260)
    for name in ("x", "w"):
        no(INVALID, f"null {name}", **{name: None})
        no(INVALID, "aligned to their elements", **{name: 257})
    no(INVALID, "stride", xs=-64)
    no(INVALID, "stride", ws_=-64)
    no(INVALID, "aligned", gate=258)
    if bwd:
        no(UNSUPPORTED, "dweight", dwt=FP16)
        no(INVALID, "null dy", dy=None)
        no(INVALID, "stride", dxs=63)
        no(INVALID, "stride", dws=63)
        no(INVALID, "aligned", dx=257)
        no(INVALID, "aligned", dw=258)
        no(INVALID, "kept", kept=None)
        no(INVALID, "kept", kept=None, act=0)
        no(INVALID, "aligned", kept=257)
        size = L.load().saf3r_linear_bwd_workspace_bytes
        need = size(3, 64, 32, 4)
        assert need > size(3, 64, 32, 0) > 0 and size(0, 64, 32, 7) == 0 and size(-1, 64, 32, 0) == -1
        assert size(3, 64, 0, 0) == -1 and size(3, 60, 32, 7) > size(3, 60, 32, 4) and size(87936, 1024, 4096, 4) > 2 ** 29
        no(INVALID, "workspace", nbytes=need - 1)
        no(INVALID, "workspace", wsp=None)
        no(INVALID, "16-byte", wsp=264)
        no(INVALID, "workspace", x=258, nbytes=need)  # (a copy of x)
        no(INVALID, "workspace", k=60, nbytes=need)
    else:
        no(INVALID, "null y", y=None)
        no(INVALID, "stride", ys=31)
        no(INVALID, "stride", ks=31)
        no(INVALID, "stride", rs=-32)
        no(INVALID, "aligned", bias=258)
        no(INVALID, "aligned", kept=257)
        size = L.load().saf3r_linear_fwd_workspace_bytes
        assert size(3, 64, 32, 1, 9, 0) == 0 and size(3, 60, 32, 0, 0, 1) > 0
        assert size(3, 60, 32, 0, 0, 3) > size(3, 60, 32, 0, 0, 2) > 0
        assert size(0, 64, 32, 0, 0, 3) == 0 and size(3, 0, 32, 0, 0, 0) == -1 and size(130, 4096, 64, 0, 0, 0) > 0
        no(INVALID, "workspace", k=60, nbytes=0)
        no(INVALID, "workspace", x=258, wsp=None)
        assert linear(L, rows=0, x=None, y=None) == 0


def residual(L, bwd=False, x=256, xs=64, xt=BF16, br=256, bs=64, yt=BF16, rows=3, dim=64, gate=256, w=256, b=256, pt=FP32,
             drop=100, state=256, eps=1e-5, h=256, hs=64, y=256, ys=64, mean=256, rstd=256, dh=256, dhs=64, dy=256, dys=64,
             dx=256, dxs=64, dbr=256, dbs=64, dg=256, dw=256, db=256, ws=256, nbytes=1 << 20):
    lib = L.load()
    if bwd:
        return lib.saf3r_residual_norm_bwd(dh, dhs, dy, dys, yt, h, hs, xt, br, bs, rows, dim, mean, rstd, gate, w, pt, drop,
                                           state, dx, dxs, dbr, dbs, dg, dw, db, ws, nbytes, None)
    return lib.saf3r_residual_norm_fwd(x, xs, xt, br, bs, yt, rows, dim, gate, w, b, pt, drop, state, eps, h, hs, y, ys, mean,
                                       rstd, None)


@pytest.mark.parametrize("bwd", [False, True])
def test_residual_norm(L, bwd):
    def no(code, text, **kw):
        refused(L, residual(L, bwd, **kw), code, text)
    no(INVALID, "sizes", rows=-1)
    no(INVALID, "sizes", dim=0)
    no(UNSUPPORTED, "at most 8192", dim=8193)
    no(UNSUPPORTED, "too many rows", rows=1 << 40)
    no(INVALID, "element type", xt=5)
    no(INVALID, "element type", pt=3)
    no(UNSUPPORTED, "keep their type", yt=FP32)
    no(UNSUPPORTED, "16-bit type", pt=FP16)
    no(UNSUPPORTED, "16-bit type", xt=FP32, yt=FP32, pt=BF16)
    for drop in (-1, 65537):
        no(INVALID, "65536 times", drop=drop)
    no(INVALID, "state", state=None)
    names = ("dy", "h", "mean", "rstd", "dx") if bwd else ("x", "br", "h", "y", "mean", "rstd")
    for name in names:
        no(INVALID, "null", **{name: None})
    if bwd:
        no(INVALID, "branch", br=None)
        no(INVALID, "aligned", dh=257)
        no(INVALID, "aligned", dbr=257)
        no(INVALID, "stride", dxs=63)
        no(INVALID, "stride", dbs=63)
        no(INVALID, "stride", dys=-64)
        size = L.load().saf3r_residual_norm_bwd_workspace_bytes
        need = size(3, 64)
        assert need > 0 and size(3, 8193) == -1 and size(-1, 64) == -1
        no(INVALID, "workspace", nbytes=need - 1)
        no(INVALID, "workspace", ws=None)
        no(INVALID, "16-byte", ws=264)
    else:
        no(INVALID, "eps", eps=-1e-5)
        no(INVALID, "eps", eps=float("nan"))
        no(INVALID, "aligned", x=257)
        no(INVALID, "stride", hs=63)
        no(INVALID, "stride", ys=63)
        no(INVALID, "stride", bs=-64)
        no(UNSUPPORTED, "too many rows for one launch", rows=(1 << 24) * 32)
        assert residual(L, rows=0, x=None) == 0


def test_dropout(L):
    def call(x=256, xs=64, type=BF16, rows=3, dim=64, drop=100, state=256, y=256, ys=64):
        return L.load().saf3r_dropout(x, xs, type, rows, dim, drop, state, y, ys, None)
    refused(L, call(rows=-1), INVALID, "sizes")
    refused(L, call(dim=0), INVALID, "sizes")
    refused(L, call(rows=1 << 40), UNSUPPORTED, "too many rows")
    refused(L, call(type=4), INVALID, "element type")
    refused(L, call(drop=65537), INVALID, "65536 times")
    refused(L, call(drop=-1), INVALID, "65536 times")
    refused(L, call(state=None), INVALID, "state")
    refused(L, call(state=None, drop=0), INVALID, "state")
    refused(L, call(x=None), INVALID, "null")
    refused(L, call(y=None), INVALID, "null")
    refused(L, call(x=257), INVALID, "aligned")
    refused(L, call(xs=-1), INVALID, "stride")
    refused(L, call(ys=63), INVALID, "stride")
    assert call(rows=0, x=None) == 0


@pytest.mark.parametrize("name", ("saf3r_linear_fwd", "saf3r_linear_bwd", "saf3r_residual_norm_fwd",
                                  "saf3r_residual_norm_bwd", "saf3r_dropout"))
def test_injected_failures(L, monkeypatch, name):
    fn = getattr(L.load(), name)

    def call():
        return fn(*[None if t is ctypes.c_void_p else 0 for t in fn.argtypes])
    for which in (name, "all"):
        monkeypatch.setenv("SAF3R_FAULT_INJECT", which)
        assert call() == 4 and name.encode() in L.load().saf3r_last_error()
    monkeypatch.setenv("SAF3R_FAULT_INJECT", name + "x")
    assert call() == 1


def test_tensors_that_are_not_on_a_gpu(pkg):
    ops = import_module(pkg.__name__ + ".ops")
    t, s = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4)
    for call in (lambda: ops.linear_fwd(t, t), lambda: ops.linear_bwd(t, t, t), lambda: ops.residual_norm_fwd(t, t),
                 lambda: ops.residual_norm_bwd(t, t, t, s, s, t), lambda: ops.dropout(t, 0.5, torch.zeros(2).long())):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_generator(pkg):
    """The tests' generator against the published known answers of Philox4x32 with ten rounds."""
    import block_ref as R
    answers = [((0,) * 4, (0,) * 2, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
               ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
               ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
                (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))]
    for counter, key, want in answers:
        assert tuple(int(w) for w in R.philox(counter, key)) == want
