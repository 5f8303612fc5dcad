"""Refusals of the token-row entry points: every check of sizes, types, alignment and nulls answers before the
first CUDA call, so the pointers here are never read and the answers are the same with and without a GPU."""
import pytest

import fenix_b200 as fx

F32, F16, BF16, E4M3 = 0, 1, 2, 3
P, Q, R, S = 0x10000, 0x20000, 0x30000, 0x40000  # aligned addresses that no call gets to read


def norm(**kw):
    a = dict(x=P, xt=BF16, rows=4, cols=64, xs=64, r=None, rt=BF16, rs=64, s=None, ss=64, w=None, wt=BF16, eps=1e-6,
             y=Q, yt=BF16, ys=64, scale=None, mode=0, stream=None)
    assert set(kw) <= set(a)
    return fx.lib().fx_rms_norm(*{**a, **kw}.values())


def linear(**kw):
    a = dict(x=P, xt=BF16, rows=4, xs=128, sc=None, mode=0, codes=Q, scales=R, st=F16, zeros=None, n=8, k=128, group=32,
             bias=None, y=S, yt=BF16, ys=8, stream=None)
    assert set(kw) <= set(a)
    return fx.lib().fx_w4_linear(*{**a, **kw}.values())


def quantize(**kw):
    a = dict(w=P, wt=F32, n=8, k=128, ws=128, group=32, codes=Q, scales=R, st=F16, zeros=None, stream=None)
    assert set(kw) <= set(a)
    return fx.lib().fx_w4_quantize(*{**a, **kw}.values())


def dequantize(**kw):
    a = dict(codes=Q, scales=R, st=F16, zeros=None, n=8, k=128, group=32, w=P, wt=F32, ws=128, stream=None)
    assert set(kw) <= set(a)
    return fx.lib().fx_w4_dequantize(*{**a, **kw}.values())


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=1 << 30), dict(cols=0), dict(cols=32769, xs=0, rs=0, ss=0, ys=0), dict(eps=0.0),
    dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(xt=E4M3), dict(xt=4), dict(xt=-1),
    dict(rt=E4M3), dict(wt=E4M3), dict(yt=7), dict(yt=E4M3), dict(yt=E4M3, mode=2), dict(yt=E4M3, scale=S, mode=3),
    dict(mode=2, scale=S), dict(mode=1, scale=S), dict(xs=63), dict(rs=1), dict(ss=63), dict(ys=63), dict(ys=-64),
    dict(xs=1 << 30), dict(x=None), dict(y=None), dict(x=P + 1), dict(y=Q + 1), dict(r=R + 1), dict(s=S + 1),
    dict(w=S + 1), dict(yt=E4M3, scale=S + 2, mode=2), dict(y=P, yt=F16), dict(y=P, xs=72), dict(s=P, rt=F32),
    dict(s=P, ss=72), dict(r=R, s=R, ss=72), dict(s=S, y=S), dict(r=S, y=S)])
def test_rms_norm_refuses(kw):
    assert norm(**kw) == fx.FX_INVALID_ARGUMENT
    assert fx.lib().fx_last_error().startswith(b"fx_rms_norm: ")


W4_BAD = [dict(n=-1), dict(n=1 << 30), dict(k=0), dict(k=-128), dict(group=0), dict(group=-32), dict(group=16),
          dict(group=48), dict(k=120), dict(group=256), dict(k=160, group=64), dict(st=E4M3), dict(st=9),
          dict(codes=None), dict(scales=None), dict(codes=Q + 8), dict(scales=R + 1), dict(scales=R + 2, st=F32)]


@pytest.mark.parametrize("kw", W4_BAD + [
    dict(rows=-1), dict(rows=1 << 30), dict(xt=F32), dict(xt=4), dict(yt=F32), dict(yt=E4M3), dict(xt=E4M3),
    dict(xt=E4M3, mode=2), dict(xt=E4M3, mode=3, sc=P), dict(mode=2, sc=P), dict(xs=127), dict(ys=7), dict(ys=1 << 31),
    dict(x=None), dict(y=None), dict(x=P + 1), dict(y=S + 1), dict(xt=E4M3, mode=1, sc=P + 2), dict(bias=P + 2),
    dict(y=P)])
def test_w4_linear_refuses(kw):
    assert linear(**kw) == fx.FX_INVALID_ARGUMENT
    assert fx.lib().fx_last_error().startswith(b"fx_w4_linear: ")


@pytest.mark.parametrize("kw", W4_BAD + [dict(wt=E4M3), dict(ws=127), dict(w=None), dict(w=P + 2)])
def test_w4_quantize_and_dequantize_refuse(kw):
    assert quantize(**kw) == fx.FX_INVALID_ARGUMENT
    assert fx.lib().fx_last_error().startswith(b"fx_w4_quantize: ")
    assert dequantize(**kw) == fx.FX_INVALID_ARGUMENT
    assert fx.lib().fx_last_error().startswith(b"fx_w4_dequantize: ")


def test_no_rows_is_no_error():
    assert norm(rows=0, x=None, y=None) == fx.FX_OK
    assert linear(rows=0, x=None, y=None) == fx.FX_OK
    assert linear(n=0, codes=None, scales=None, y=None) == fx.FX_OK
    assert quantize(n=0, w=None, codes=None, scales=None) == fx.FX_OK
    assert dequantize(n=0, w=None, codes=None, scales=None) == fx.FX_OK


def test_python_names_of_types_and_modes():
    with pytest.raises(KeyError):
        fx.rms_norm_dev(P, Q, 1, 8, x_type="f64")
    with pytest.raises(KeyError):
        fx.w4_linear_dev(P, Q, 1, 8, 32, 32, R, S, x_scale_mode="column")
    with pytest.raises(fx.FxError) as e:
        fx.w4_linear_dev(P, Q, 1, 8, 48, 32, R, S)
    assert e.value.code == fx.FX_INVALID_ARGUMENT and "group" in str(e.value)
