"""Calls of the training operators that are refused, with the reason, before anything is launched (CPU: the C entries
with addresses that are never read; the wrappers' checks of tensors that are not on a GPU)."""
import ctypes
from importlib import import_module

import pytest
import torch

FP32, BF16, FP16 = 0, 1, 2


@pytest.fixture(scope="module")
def L(pkg):
    return import_module(pkg.__name__ + "._lib")


def heads(L, ptr=256, clip=640, token=64, group=64, head=64):
    return ctypes.byref(L.Heads(ptr, clip, token, group, head))


def refused(L, rc, code, text):
    msg = L.load().saf3r_last_error().decode()
    assert rc == code and text in msg, (rc, msg)


INVALID, UNSUPPORTED = 1, 2


def attn_fwd(L, q=None, k=None, v=None, clips=1, frames=2, tokens=5, n=1, patterns=(0,), scale=0.125, out=None,
             rest=None, lse=256):
    h = heads(L)
    pat = (ctypes.c_int32 * max(1, len(patterns)))(*patterns) if patterns is not None else None
    return L.load().saf3r_frame_attn_fwd(q or h, k or h, v or h, clips, frames, tokens, n, pat, None, scale, out or h,
                                         rest, lse, None)


def attn_bwd(L, clips=1, frames=2, tokens=5, n=1, patterns=(0,), scale=0.125, ws=256, nbytes=1 << 20, **t):
    h = heads(L)
    pat = (ctypes.c_int32 * len(patterns))(*patterns)
    g = lambda name: t.get(name, h)  # noqa: E731
    return L.load().saf3r_frame_attn_bwd(g("dout"), g("q"), g("k"), g("v"), g("out"), t.get("rest"), t.get("lse", 256),
                                         clips, frames, tokens, n, pat, None, scale, g("dq"), g("dk"), g("dv"), ws,
                                         nbytes, None)


@pytest.mark.parametrize("call", [attn_fwd, attn_bwd])
def test_attention_sizes_and_patterns(L, call):
    refused(L, call(L, frames=0), INVALID, "sizes")
    refused(L, call(L, tokens=0), INVALID, "sizes")
    refused(L, call(L, clips=-1), INVALID, "sizes")
    refused(L, call(L, n=0), INVALID, "num_heads")
    refused(L, call(L, n=65, patterns=(0,) * 65), UNSUPPORTED, "at most 64")
    refused(L, call(L, frames=1 << 16, tokens=1 << 16), UNSUPPORTED, "31 bits")
    for p in (3, 4, 7, 8, 9):
        refused(L, call(L, patterns=(p,)), UNSUPPORTED, "pattern")
    for p in (-1, 10):
        refused(L, call(L, patterns=(p,)), INVALID, "pattern")
    for s in (0.0, -1.0, float("inf"), float("nan")):
        refused(L, call(L, scale=s), INVALID, "scale")
    assert call(L, clips=0) == 0


def test_attention_tensors(L):
    refused(L, attn_fwd(L, patterns=None), INVALID, "null patterns")
    for name in ("q", "k", "v", "out"):
        refused(L, attn_fwd(L, **{name: heads(L, ptr=None)}), INVALID, "null")
        refused(L, attn_fwd(L, **{name: heads(L, ptr=264)}), INVALID, "aligned")
        for stride in ("clip", "token", "head"):
            refused(L, attn_fwd(L, **{name: heads(L, **{stride: 68})}), INVALID, "multiple of 8")
    refused(L, attn_fwd(L, rest=heads(L, ptr=None)), INVALID, "out_rest")
    refused(L, attn_fwd(L, rest=heads(L, ptr=258)), INVALID, "aligned")
    refused(L, attn_fwd(L, lse=None), INVALID, "null")
    refused(L, attn_fwd(L, lse=258), INVALID, "aligned")
    for name in ("dout", "q", "k", "v", "out", "dq", "dk", "dv"):
        refused(L, attn_bwd(L, **{name: heads(L, ptr=None)}), INVALID, "null")
        refused(L, attn_bwd(L, **{name: heads(L, token=60)}), INVALID, "multiple of 8")
    refused(L, attn_bwd(L, lse=None), INVALID, "null")
    size = L.load().saf3r_frame_attn_bwd_workspace_bytes
    need = size(1, 2, 5, 1)
    assert need > 0 and size(0, 2, 5, 1) == 0 and size(1, 0, 5, 1) == -1 and size(1, 2, 5, 65) == -1
    assert size(1, 1 << 16, 1 << 16, 1) == -1 and size(7, 1000, 1374, 64) > 2 ** 31
    refused(L, attn_bwd(L, nbytes=need - 1), INVALID, "workspace")
    refused(L, attn_bwd(L, ws=None), INVALID, "workspace")
    refused(L, attn_bwd(L, ws=264), INVALID, "16-byte")


@pytest.mark.parametrize("call", [attn_fwd, attn_bwd])
def test_attention_scale_range(L, call):
    for s in (1e-31, 1e31, -0.125):
        refused(L, call(L, scale=s), INVALID, "scale")


def test_attention_results_on_each_other(L):
    """Rows that are written have places of their own; rows that are read may be broadcast (not refused here: the call
    goes on to the next check)."""
    sizes = dict(clips=2, n=2, patterns=(0, 0))
    for stride in ("clip", "token", "head"):
        h = heads(L, **{stride: 0})
        refused(L, attn_fwd(L, out=h, **sizes), INVALID, "overlap")
        refused(L, attn_fwd(L, rest=h, **sizes), INVALID, "overlap")
        for name in ("dq", "dk", "dv"):
            refused(L, attn_bwd(L, **{name: h}, **sizes), INVALID, "overlap")
        for name in ("dout", "q", "k", "v", "out"):
            refused(L, attn_bwd(L, nbytes=0, **{name: h}, **sizes), INVALID, "workspace")


@pytest.mark.parametrize("bwd", [False, True])
def test_rotary_results_on_each_other(L, bwd):
    for stride in ("clip", "token", "group", "head"):
        for norm in (0, 1):
            refused(L, rotary(L, bwd, y=heads(L, **{stride: 0}), clips=2, norm=norm), INVALID, "overlap")


def test_launches_beyond_32_bits_of_threads(L):
    for call in (attn_fwd, attn_bwd):
        kw = {} if call is attn_fwd else {"nbytes": 1 << 40}
        refused(L, call(L, clips=1 << 23, frames=1, tokens=1, **kw), UNSUPPORTED, "too many row tiles")
    refused(L, norm(L, rows=(1 << 24) * 32), UNSUPPORTED, "too many rows for one launch")


def rotary(L, bwd=False, x=None, y=None, dy=None, type=BF16, clips=1, tokens=3, groups=2, n=2, dim=64, pos=256, pos64=1,
           axes=2, cos=256, sin=256, positions=9, rot=64, inter=0, norm=1, w=256, b=256, pt=FP32, eps=1e-5, ws=256,
           nbytes=1 << 20):
    h = heads(L)
    lib = L.load()
    if bwd:
        return lib.saf3r_head_rotary_bwd(dy or h, x or h, type, clips, tokens, groups, n, dim, pos, pos64, axes, cos, sin,
                                         positions, rot, inter, norm, w, pt, eps, y or h, 256, 256, ws, nbytes, None)
    return lib.saf3r_head_rotary_fwd(x or h, type, clips, tokens, groups, n, dim, pos, pos64, axes, cos, sin, positions,
                                     rot, inter, norm, w, b, pt, eps, y or h, None)


@pytest.mark.parametrize("bwd", [False, True])
def test_rotary(L, bwd):
    def no(code, text, **kw):
        refused(L, rotary(L, bwd, **kw), code, text)
    for kw in ({"clips": -1}, {"tokens": -1}, {"groups": 0}, {"n": 0}, {"dim": 0}):
        no(INVALID, "sizes", **kw)
    for dim in (130, 63, 256):
        no(UNSUPPORTED, "rows of", dim=dim)
    no(UNSUPPORTED, "groups", groups=65)
    no(UNSUPPORTED, "too many rows", clips=1 << 20, tokens=1 << 12)
    no(UNSUPPORTED, "too many rows", clips=1 << 60, tokens=1 << 12)
    no(INVALID, "element type", type=3)
    no(INVALID, "element type", pt=-1)
    no(UNSUPPORTED, "16-bit type", pt=FP16)
    no(UNSUPPORTED, "16-bit type", type=FP32, pt=BF16)
    no(INVALID, "positions", sin=None)
    no(INVALID, "positions", pos=None)
    no(INVALID, "positions", positions=0)
    for kw in ({"axes": 0}, {"axes": 9}, {"rot": 0}, {"rot": 66}, {"rot": 62}, {"rot": 30}):
        no(INVALID, "axes", **kw)
    no(INVALID, "aligned", pos=260)
    no(INVALID, "aligned", cos=258)
    no(INVALID, "eps", eps=-1.0)
    no(INVALID, "eps", eps=float("nan"))
    no(INVALID, "null", x=heads(L, ptr=None))
    no(INVALID, "null", y=heads(L, ptr=None))
    no(INVALID, "aligned", x=heads(L, ptr=257))
    if bwd:
        no(INVALID, "null", dy=heads(L, ptr=None))
        need = L.load().saf3r_head_rotary_bwd_workspace_bytes(1, 3, 2, 2, 64)
        no(INVALID, "workspace", nbytes=need - 1)
        no(INVALID, "workspace", ws=None)
        no(INVALID, "16-byte", ws=264)
        assert L.load().saf3r_head_rotary_bwd_workspace_bytes(1, 3, 2, 2, 63) == -1
    else:
        assert rotary(L, clips=0) == 0 and rotary(L, tokens=0, pos=None) == 0


def norm(L, bwd=False, x=256, xs=64, xt=BF16, rows=3, dim=64, w=256, b=256, pt=FP32, eps=1e-5, y=256, ys=64, yt=BF16,
         mean=256, rstd=256, dy=256, dys=64, ws=256, nbytes=1 << 20):
    lib = L.load()
    if bwd:
        return lib.saf3r_layer_norm_bwd(dy, dys, yt, x, xs, xt, rows, dim, mean, rstd, w, pt, y, ys, 256, 256, ws, nbytes,
                                        None)
    return lib.saf3r_layer_norm_fwd(x, xs, xt, rows, dim, w, b, pt, eps, y, ys, yt, mean, rstd, None)


@pytest.mark.parametrize("bwd", [False, True])
def test_layer_norm(L, bwd):
    def no(code, text, **kw):
        refused(L, norm(L, bwd, **kw), code, text)
    no(INVALID, "sizes", rows=-1)
    no(INVALID, "sizes", dim=0)
    no(UNSUPPORTED, "at most 8192", dim=8193)
    no(UNSUPPORTED, "too many rows", rows=1 << 40)
    no(INVALID, "element type", xt=5)
    no(INVALID, "element type", pt=3)
    no(UNSUPPORTED, "keep their type", yt=FP32)
    no(UNSUPPORTED, "keep their type", yt=FP16)
    no(UNSUPPORTED, "16-bit type", pt=FP16)
    no(UNSUPPORTED, "16-bit type", xt=FP32, yt=FP32, pt=BF16)
    for name in ("x", "y", "mean", "rstd") + (("dy",) if bwd else ()):
        no(INVALID, "null", **{name: None})
    no(INVALID, "aligned", x=257)
    no(INVALID, "stride", xs=-64)
    no(INVALID, "stride", ys=63)
    if bwd:
        need = L.load().saf3r_layer_norm_bwd_workspace_bytes(3, 64)
        no(INVALID, "workspace", nbytes=need - 1)
        no(INVALID, "workspace", ws=None)
        no(INVALID, "16-byte", ws=264)
        assert L.load().saf3r_layer_norm_bwd_workspace_bytes(3, 8193) == -1
    else:
        no(INVALID, "eps", eps=-1e-5)
        assert norm(L, rows=0, x=None) == 0


ENTRIES = ("saf3r_frame_attn_fwd", "saf3r_frame_attn_bwd", "saf3r_head_rotary_fwd", "saf3r_head_rotary_bwd",
           "saf3r_layer_norm_fwd", "saf3r_layer_norm_bwd")


@pytest.mark.parametrize("name", ENTRIES)
def test_injected_failures(L, monkeypatch, name):
    fn = getattr(L.load(), name)

    def call():
        return fn(*[None if t is ctypes.c_void_p or hasattr(t, "contents") else 0 for t in fn.argtypes])
    for which in (name, "all"):
        monkeypatch.setenv("SAF3R_FAULT_INJECT", which)
        assert call() == 4 and name.encode() in L.load().saf3r_last_error()
    monkeypatch.setenv("SAF3R_FAULT_INJECT", name + "x")
    assert call() == 1


def test_tensors_that_are_not_on_a_gpu(pkg):
    ops = import_module(pkg.__name__ + ".ops")
    t = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    lse = torch.zeros(1, 2, 4)
    for call in (lambda: ops.frame_attn_fwd(t, t, t, [0, 0]),
                 lambda: ops.frame_attn_bwd(t, t, t, t, t, lse, [0, 0]),
                 lambda: ops.head_rotary_fwd(t[:, :, None], norm=True),
                 lambda: ops.head_rotary_bwd(t[:, :, None], t[:, :, None], norm=True),
                 lambda: ops.layer_norm_fwd(t),
                 lambda: ops.layer_norm_bwd(t, t, lse, lse)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_rotary_tables(pkg):
    ops = import_module(pkg.__name__ + ".ops")
    cos, sin = ops.rotary_tables(50, 32, base=100.0, device="cpu")
    ref = ops.rope_tables(50, 100.0, device="cpu")  # the forward path's tables, from fp32 angles of at most 50
    assert cos.shape == (50, 16) and (cos - ref[0]).abs().max() < 50 * 2.0 ** -23 and (sin - ref[1]).abs().max() < 50 * 2.0 ** -23
    pos = torch.arange(50, dtype=torch.float64)[:, None]
    inv = 100.0 ** -(torch.arange(0, 32, 2, dtype=torch.float64) / 32)
    lin = ops.rotary_tables(50, 32, 100.0, "linear", 4.0, device="cpu")
    assert (lin[1].double() - (pos / 4 * inv).sin()).abs().max() < 2.0 ** -24
    ntk = ops.rotary_tables(50, 32, 100.0, "ntk", 4.0, device="cpu")
    ang = pos * (100.0 * 4.0 ** (32 / 30)) ** -(torch.arange(0, 32, 2, dtype=torch.float64) / 32)
    assert (ntk[1].double() - ang.sin()).abs().max() < 2.0 ** -24
    assert torch.equal(ntk[0][:, 0], cos[:, 0])  # the fastest pair keeps its angles
    assert abs(float(ang[1, -1] / inv[-1]) - 0.25) < 1e-12  # the slowest one's are a fourth
    for bad in (dict(positions=0, section=32), dict(positions=4, section=3), dict(positions=4, section=0),
                dict(positions=4, section=32, base=0.0), dict(positions=4, section=32, base=float("inf")),
                dict(positions=4, section=32, factor=-1.0), dict(positions=4, section=32, scaling="other"),
                dict(positions=4, section=2, scaling="ntk", factor=2.0)):
        with pytest.raises(ValueError):
            ops.rotary_tables(device="cpu", **bad)


def test_kept_tables_of_an_inference_run(pkg):
    """Tables that a run without gradients made first can be saved by a training step."""
    ops = import_module(pkg.__name__ + ".ops")
    with torch.inference_mode():
        kept = ops.rope_tables(7, 77.0, "cpu")
    assert not any(t.is_inference() for t in kept)
    x = torch.ones(7, 16, requires_grad=True)
    (x * ops.rope_tables(7, 77.0, "cpu")[0]).sum().backward()
