"""What the 8-bit operators refuse, and that they refuse it before they touch the device or the context.

These run without a GPU: the context handed in is a dummy, so a call that got past its checks would not
return one of the codes asserted here.  Addresses are made up; none is read.
"""
import ctypes

import pytest

import glacier_paged as gp

BAD, UNSUPPORTED, OK = gp.GSP_E_INVALID_ARG, gp.GSP_E_UNSUPPORTED, gp.GSP_OK
CTX = ctypes.cast(ctypes.create_string_buffer(1), ctypes.c_void_p)
NAN, INF = float("nan"), float("inf")
X, R, W, S, Y, C, K = (i << 32 for i in range(1, 8))  # far apart


def norm(**kw):
    a = dict(rows=4, dim=64, x=X, residual=R, weight=W, eps=1e-6, sum=S, y=Y, codes=C, scale=K, ctx=CTX)
    a.update(kw)
    return gp.load().gsp_rms_norm(a["ctx"], a["rows"], a["dim"], a["x"], a["residual"], a["weight"], a["eps"],
                                  a["sum"], a["y"], a["codes"], a["scale"])


@pytest.mark.parametrize("kw", [
    dict(ctx=None), dict(rows=-1), dict(dim=0), dict(dim=-64), dict(eps=-1e-6), dict(eps=NAN), dict(eps=INF),
    dict(x=None), dict(weight=None), dict(codes=None), dict(scale=None), dict(sum=None, y=None, codes=None, scale=None),
    dict(residual=None), dict(x=X + 2), dict(residual=R + 1), dict(weight=W + 2), dict(sum=S + 2), dict(y=Y + 1),
    dict(scale=K + 2),
    dict(sum=X + 4), dict(y=R - 4), dict(y=S), dict(codes=X), dict(codes=S + 4), dict(scale=C + 252), dict(sum=W),
    dict(y=W - 4), dict(scale=R + 4 * 255), dict(y=X, sum=X),
], ids=str)
def test_norm_refuses(kw):
    assert norm(**kw) == BAD and gp.load().gsp_last_error()


def test_norm_of_no_rows_is_nothing():
    assert norm(rows=0) == OK
    assert norm(rows=0, x=None, weight=None) == OK


def quantize(**kw):
    a = dict(act=gp.ACT_SILU_MUL, rows=4, dim=64, stride=128, a=X, b=X + 256, codes=C, scale=K, ctx=CTX)
    a.update(kw)
    return gp.load().gsp_quantize_fp8(a["ctx"], a["act"], a["rows"], a["dim"], a["stride"], a["a"], a["b"], a["codes"],
                                      a["scale"])


@pytest.mark.parametrize("kw", [
    dict(ctx=None), dict(act=2), dict(act=-1), dict(rows=-1), dict(dim=0), dict(stride=63), dict(stride=-128),
    dict(stride=(1 << 63) - 1), dict(a=None), dict(b=None), dict(codes=None), dict(scale=None), dict(act=gp.ACT_NONE),
    dict(a=X + 1), dict(b=X + 258), dict(scale=K + 1), dict(codes=X), dict(codes=X + 4 * (3 * 128 + 64) - 1, b=R),
    dict(scale=X + 512), dict(scale=C), dict(b=C - 4),
], ids=str)
def test_quantize_refuses(kw):
    assert quantize(**kw) == BAD and gp.load().gsp_last_error()


def test_quantize_of_no_rows_is_nothing():
    assert quantize(rows=0) == OK


def matmul(**kw):
    a = dict(w_type=gp.WTYPE_Q4_0, w=W, x=X, scale=K, y=Y, in_dim=512, out_dim=48, batch=5, ctx=CTX)
    a.update(kw)
    return gp.load().gsp_matmul_batch_fp8(a["ctx"], a["w_type"], a["w"], a["x"], a["scale"], a["y"], a["in_dim"],
                                          a["out_dim"], a["batch"])


@pytest.mark.parametrize("kw", [
    dict(ctx=None), dict(in_dim=-64), dict(out_dim=-1), dict(batch=-1), dict(w=None), dict(x=None), dict(scale=None),
    dict(y=None), dict(w=W + 2), dict(x=X + 8), dict(scale=K + 2), dict(y=Y + 2),
    dict(y=X), dict(y=X + 5 * 512 - 4), dict(y=W + 48 * 288 - 4), dict(y=K + 16), dict(y=K - 4 * 48 * 5 + 4),
], ids=str)
def test_matmul_refuses(kw):
    assert matmul(**kw) == BAD and gp.load().gsp_last_error()


@pytest.mark.parametrize("kw", [
    dict(w_type=gp.WTYPE_F32), dict(w_type=gp.WTYPE_Q8_0), dict(w_type=gp.WTYPE_Q6_K), dict(w_type=99),
    dict(in_dim=0), dict(in_dim=32), dict(in_dim=480), dict(w_type=gp.WTYPE_Q4_K, in_dim=320),
    dict(out_dim=(1 << 24) + 1), dict(out_dim=(1 << 31) - 1, batch=(1 << 31) - 1),
], ids=str)
def test_matmul_unsupported(kw):
    assert matmul(**kw) == UNSUPPORTED and gp.load().gsp_last_error()


def test_matmul_of_nothing_is_nothing():
    assert matmul(batch=0) == OK
    assert matmul(out_dim=0) == OK


def test_mrope_without_context_or_pool():
    spec = gp.MRope(1e4, [4, 6, 6]).spec(32)
    f = gp.load().gsp_mrope_write_step
    assert f(None, None, 0, 1, ctypes.byref(spec), X, X, 0, Y, X, 0, X, 0) == BAD
    assert f(CTX, None, 0, 1, ctypes.byref(spec), X, X, 0, Y, X, 0, X, 0) == BAD


def test_mrope_takes_at_most_four_axes():
    with pytest.raises(ValueError):
        gp.MRope(1e4, [4, 4, 4, 2, 2])
