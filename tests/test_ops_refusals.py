"""Refusals of the handle-free operators (lcn_orthogonalize, lcn_muon_update, lcn_int8_linear,
lcn_int8_quantize_weight): every bad call is an error before anything is launched, so all of this
runs without a GPU -- the pointers below are addresses that nothing reads."""
import ctypes

import pytest
import torch

from lcn_amd import native, ops

F32, F64, BF16, F16 = 0, 1, 2, 3
A, B, C, WS = 1 << 32, 2 << 32, 3 << 32, 8 << 32
BIG = 1 << 40
COEF = (ctypes.c_float * 3)(3.4445, -4.775, 2.0315)


@pytest.fixture(scope="module")
def lib():
    return native.load_library()


def _orth(lib, **kw):
    a = dict(dtype=F32, batch=2, rows=8, cols=16, inp=A, ib=128, ir=16, out=B, ob=128, orow=16, steps=5, coef=COEF,
             eps=1e-7, ws=WS, wsb=BIG)
    a.update(kw)
    return lib.lcn_orthogonalize(0, None, a["dtype"], a["batch"], a["rows"], a["cols"], a["inp"], a["ib"], a["ir"],
                                 a["out"], a["ob"], a["orow"], a["steps"], a["coef"], a["eps"], a["ws"], a["wsb"])


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=F64), "dtype"), (dict(dtype=9), "dtype"), (dict(batch=-1), "negative"), (dict(rows=-1), "negative"),
    (dict(batch=65536), "65535"), (dict(rows=70000, ir=70000), "too large"), (dict(rows=65536, cols=65536), "too large"),
    (dict(batch=60000, rows=512, cols=512), "too large"),
    (dict(steps=0), "steps"), (dict(steps=65), "steps"), (dict(coef=None), "coefficients"),
    (dict(coef=(ctypes.c_float * 3)(1, float("nan"), 0)), "coefficients"), (dict(eps=0.0), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(inp=None), "null"), (dict(out=None), "null"), (dict(ws=None), "workspace"),
    (dict(ws=WS + 64), "aligned"), (dict(wsb=100), "needed"), (dict(inp=A + 2), "aligned"), (dict(out=B + 1), "aligned"),
    (dict(ir=-16), "strides"), (dict(ib=-1), "strides"), (dict(orow=15), "overlap"), (dict(ob=16), "overlap"),
    (dict(out=A + 64), "overlaps the input"), (dict(out=A, orow=32, ob=256), "overlaps the input"),
    (dict(inp=WS + 256), "workspace overlaps"), (dict(out=WS + 512), "workspace overlaps"),
    (dict(ib=1 << 62), "strides"),
])
def test_orthogonalize_refuses(lib, kw, word):
    assert _orth(lib, **kw) == -1
    assert word in lib.lcn_last_error(None).decode()


def test_empty_batches_are_fine(lib):
    assert _orth(lib, batch=0, inp=None, out=None, ws=None, wsb=0) == 0
    assert _orth(lib, rows=0) == 0 and _orth(lib, cols=0) == 0
    assert lib.lcn_orthogonalize_workspace(0, 8, 8) == 0
    assert lib.lcn_orthogonalize_workspace(1, 8, -1) == -1
    assert lib.lcn_int8_linear_workspace(0, 8, 8) == 0
    assert lib.lcn_int8_linear_workspace(4, 131073, 8) == -1


def _muon(lib, **kw):
    a = dict(dtype=F32, batch=2, rows=8, cols=16, p=A, pb=128, pr=16, m=B, mb=128, mr=16, g=C, gb=128, gr=16, lr=1e-3,
             lr_dev=None, scale=1.0, beta=0.95, decay=0.0, steps=5, coef=COEF, eps=1e-7, ws=WS, wsb=BIG)
    a.update(kw)
    return lib.lcn_muon_update(0, None, a["dtype"], a["batch"], a["rows"], a["cols"], a["p"], a["pb"], a["pr"], a["m"],
                               a["mb"], a["mr"], a["g"], a["gb"], a["gr"], a["lr"], a["lr_dev"], a["scale"], a["beta"],
                               1, a["decay"], a["steps"], a["coef"], a["eps"], a["ws"], a["wsb"])


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=F64), "grad_dtype"), (dict(lr=float("nan")), "finite"), (dict(scale=float("inf")), "finite"),
    (dict(decay=float("nan")), "finite"), (dict(beta=1.0), "beta"), (dict(beta=-0.1), "beta"),
    (dict(beta=float("nan")), "beta"), (dict(p=None), "null"), (dict(m=None), "null"), (dict(g=None), "null"),
    (dict(p=B), "must not overlap"), (dict(g=A), "must not overlap"), (dict(g=B + 4), "must not overlap"),
    (dict(pr=8), "overlap"), (dict(mb=0), "overlap"), (dict(gr=-1), "gradient"), (dict(lr_dev=A + 2), "aligned"),
    (dict(lr_dev=A + 64), "lr_dev"), (dict(lr_dev=B), "lr_dev"), (dict(lr_dev=WS + 256), "lr_dev"),
    (dict(m=WS), "workspace overlaps"), (dict(wsb=0), "needed"), (dict(steps=-1), "steps"),
])
def test_muon_update_refuses(lib, kw, word):
    assert _muon(lib, **kw) == -1
    assert word in lib.lcn_last_error(None).decode()


def _int8(lib, **kw):
    a = dict(dtype=F32, t=40, k=32, n=16, x=A, xr=32, w=B, wr=32, s=C, b=None, out=4 << 32, orow=16, ws=WS, wsb=BIG)
    a.update(kw)
    return lib.lcn_int8_linear(0, None, a["dtype"], a["t"], a["k"], a["n"], a["x"], a["xr"], a["w"], a["wr"], a["s"],
                               a["b"], a["out"], a["orow"], a["ws"], a["wsb"])


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=F64), "dtype"), (dict(t=-1), "negative"), (dict(k=0), "k is zero"), (dict(k=131073), "131072"),
    (dict(n=(1 << 24) + 1), "too many"), (dict(t=1 << 30, n=1 << 20), "too large"), (dict(x=None), "null"),
    (dict(w=None), "null"), (dict(s=None), "null"), (dict(out=None), "null"), (dict(x=A + 2), "aligned"),
    (dict(s=C + 2), "aligned"), (dict(b=C + 1), "aligned"), (dict(xr=-1), "strides"), (dict(wr=-4), "strides"),
    (dict(orow=15), "rows overlap"), (dict(out=A + 16), "overlaps an input"), (dict(out=B), "overlaps an input"),
    (dict(out=C), "overlaps an input"), (dict(b=4 << 32), "overlaps an input"),
    (dict(k=2048, xr=2048, wr=2048, ws=None), "null workspace"), (dict(k=2048, xr=2048, wr=2048, ws=WS + 8), "256-byte"),
    (dict(k=2048, xr=2048, wr=2048, wsb=16), "needed"), (dict(k=2048, xr=2048, wr=2048, w=WS + 16), "workspace overlaps"),
])
def test_int8_linear_refuses(lib, kw, word):
    assert _int8(lib, **kw) == -1
    assert word in lib.lcn_last_error(None).decode()


def test_int8_linear_empty(lib):
    assert _int8(lib, t=0, x=None, ws=None) == 0 and _int8(lib, n=0, w=None) == 0


@pytest.mark.parametrize("args,word", [
    ((F64, 4, 8, A, 8, 1, B, C), "dtype"), ((F32, 4, 0, A, 8, 1, B, C), "k is zero"), ((F32, -4, 8, A, 8, 1, B, C), "negative"),
    ((F32, 4, 8, None, 8, 1, B, C), "null"), ((F32, 4, 8, A, -8, 1, B, C), "strides"), ((F32, 4, 8, A + 1, 8, 1, B, C), "aligned"),
    ((F32, 4, 8, A, 8, 1, A + 4, C), "overlap"), ((F32, 4, 8, A, 8, 1, B, B), "overlap"),
])
def test_quantize_weight_refuses(lib, args, word):
    assert lib.lcn_int8_quantize_weight(0, None, *args) == -1
    assert word in lib.lcn_last_error(None).decode()


def test_columns_of_one_buffer_do_not_overlap(lib):
    """An output beside its input in the same rows passes the overlap check (and only then fails, on the workspace)."""
    ok = dict(rows=8, cols=16, batch=1, inp=A, ir=64, out=A + 16 * 4, orow=64, wsb=1)
    assert _orth(lib, **ok) == -1 and "needed" in lib.lcn_last_error(None).decode()
    assert _orth(lib, **{**ok, "out": A + 15 * 4}) == -1 and "overlaps the input" in lib.lcn_last_error(None).decode()
    assert _orth(lib, **{**ok, "out": A + 49 * 4}) == -1 and "overlaps the input" in lib.lcn_last_error(None).decode()


def test_host_tensors_are_refused():
    g = torch.zeros(4, 4)
    for call in (lambda: ops.orthogonalize(g), lambda: ops.muon_update(g, g.clone(), g.clone(), lr=1e-3),
                 lambda: ops.int8_linear(g, g.to(torch.int8), g[0]), lambda: ops.quantize_weight(g),
                 lambda: ops.orthogonalize([1.0])):
        with pytest.raises(ValueError):
            call()
