"""Refusals of the 8-bit linear layer's, its quantiser's and the layer norm's entry points: every check of sizes, types,
alignment and nulls answers before the first CUDA call, so the pointers here are never read and the answers are the same with
and without a GPU."""
import pytest

import fenix_b200 as fx

F32, F16, BF16, E4M3, I8 = 0, 1, 2, 3, 4
NONE, TENSOR, ROW = 0, 1, 2
P, Q, R, S, T, V = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 0x60000  # aligned addresses that no call gets to read


def norm(**kw):
    a = dict(x=P, xt=BF16, rows=4, cols=64, xs=64, r=None, rt=BF16, rs=64, s=None, ss=64, w=None, b=None, wt=BF16, eps=1e-6,
             y=Q, yt=BF16, ys=64, mean=None, rstd=None, scale=None, mode=NONE, stream=None)
    assert set(kw) <= set(a)
    return fx.lib().fx_layer_norm(*{**a, **kw}.values())


def backward(**kw):
    a = dict(dy=P, dyt=BF16, rows=4, cols=64, ds=64, h=Q, ht=BF16, hs=64, mean=R, rstd=S, w=None, wt=BF16, dsum=None, dss=64,
             dx=T, dxt=BF16, dxs=64, dw=None, db=None, acc=0, work=None, bytes=0, stream=None)
    assert set(kw) <= set(a)
    return fx.lib().fx_layer_norm_backward(*{**a, **kw}.values())


def quantize(**kw):
    a = dict(x=P, xt=F32, rows=8, cols=128, xs=128, codes=Q, cs=128, scales=R, mode=ROW, stream=None)
    assert set(kw) <= set(a)
    return fx.lib().fx_i8_quantize(*{**a, **kw}.values())


def dequantize(**kw):
    a = dict(codes=Q, cs=128, scales=R, mode=ROW, rows=8, cols=128, y=P, yt=F32, ys=128, stream=None)
    assert set(kw) <= set(a)
    return fx.lib().fx_i8_dequantize(*{**a, **kw}.values())


def linear(**kw):
    a = dict(x=P, rows=4, xs=128, xsc=Q, mode=ROW, codes=R, cs=128, scales=S, n=8, k=128, bias=None, y=T, yt=BF16, ys=8,
             stream=None)
    assert set(kw) <= set(a)
    return fx.lib().fx_i8_linear(*{**a, **kw}.values())


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=1 << 30), dict(cols=0), dict(cols=32769, xs=0, rs=0, ss=0, ys=0), dict(eps=0.0),
    dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(xt=E4M3), dict(xt=I8), dict(xt=5), dict(xt=-1),
    dict(rt=E4M3), dict(rt=I8), dict(wt=E4M3), dict(wt=I8), dict(yt=5), dict(yt=E4M3), dict(yt=I8), dict(yt=I8, mode=ROW),
    dict(yt=E4M3, mode=ROW), dict(yt=I8, scale=S, mode=3), dict(yt=I8, scale=S), dict(mode=ROW, scale=S),
    dict(mode=TENSOR, scale=S), dict(xs=63), dict(rs=1), dict(ss=63), dict(ys=63), dict(ys=-64), dict(xs=1 << 30), dict(x=None),
    dict(y=None), dict(x=P + 1), dict(y=Q + 1), dict(r=R + 1), dict(s=S + 1), dict(w=S + 1), dict(b=S + 1), dict(mean=S + 2),
    dict(rstd=S + 2), dict(yt=I8, scale=S + 2, mode=ROW), dict(y=P, yt=F16), dict(y=P, xs=72), dict(s=P, rt=F32),
    dict(s=P, ss=72), dict(r=R, s=R, ss=72), dict(s=S, y=S), dict(r=S, y=S), dict(mean=S, rstd=S),
    dict(mean=S, yt=I8, scale=S, mode=ROW), dict(rstd=S, yt=I8, scale=S, mode=ROW)])
def test_layer_norm_refuses(kw):
    assert norm(**kw) == fx.FX_INVALID_ARGUMENT
    assert fx.lib().fx_last_error().startswith(b"fx_layer_norm: ")


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=1 << 30), dict(cols=0), dict(cols=32769, ds=0, hs=0, dss=0, dxs=0), dict(dyt=E4M3), dict(dyt=I8),
    dict(ht=E4M3), dict(ht=-1), dict(wt=I8), dict(dxt=E4M3), dict(dxt=9), dict(ds=63), dict(hs=63), dict(dss=63), dict(dxs=63),
    dict(dxs=1 << 30), dict(dx=None), dict(dy=None), dict(h=None), dict(mean=None), dict(rstd=None), dict(dy=P + 1),
    dict(h=Q + 1), dict(mean=R + 2), dict(rstd=S + 2), dict(w=V + 1), dict(dsum=V + 1), dict(dx=T + 1), dict(dw=V + 2, work=V),
    dict(db=V + 2, work=V), dict(dx=P, dxt=F32), dict(dx=P, dxs=72), dict(dx=Q, dxt=F16), dict(dx=Q, hs=72),
    dict(dsum=T, dss=72), dict(dw=V, db=V, work=V + 64, bytes=1 << 30), dict(dw=V), dict(db=V), dict(dw=V, work=V + 64),
    dict(dw=V, work=V + 64, bytes=4 * 64 * 8 - 1), dict(db=V, work=V + 68, bytes=1 << 30)])
def test_layer_norm_backward_refuses(kw):
    assert backward(**kw) == fx.FX_INVALID_ARGUMENT
    assert fx.lib().fx_last_error().startswith(b"fx_layer_norm_backward: ")


def test_layer_norm_backward_workspace():
    size = fx.layer_norm_backward_workspace
    assert size(0, 64) == 0 and size(-1, 64) == 0 and size(4, 0) == 0 and size(4, 32769) == 0 and size(1 << 30, 8) == 0
    assert size(4, 64) == 4 * 64 * 8  # a line of sums for each row at most
    for cols in (1, 1000, 4096, 8192, 32768):
        assert size(1 << 20, cols) == size(5000, cols) <= 80 << 20
        assert size(5000, cols) % (8 * cols) == 0


I8_BAD = [dict(rows=-1), dict(rows=1 << 30), dict(cols=0), dict(cols=-8), dict(cols=1 << 30), dict(cs=127), dict(cs=1 << 30),
          dict(mode=NONE), dict(mode=3), dict(codes=None), dict(scales=None), dict(scales=R + 2)]


@pytest.mark.parametrize("kw", I8_BAD + [dict(xt=E4M3), dict(xt=I8), dict(xs=127), dict(x=None), dict(x=P + 2), dict(codes=P)])
def test_i8_quantize_refuses(kw):
    assert quantize(**kw) == fx.FX_INVALID_ARGUMENT
    assert fx.lib().fx_last_error().startswith(b"fx_i8_quantize: ")


@pytest.mark.parametrize("kw", I8_BAD + [dict(yt=E4M3), dict(yt=I8), dict(ys=127), dict(y=None), dict(y=P + 2), dict(codes=P)])
def test_i8_dequantize_refuses(kw):
    assert dequantize(**kw) == fx.FX_INVALID_ARGUMENT
    assert fx.lib().fx_last_error().startswith(b"fx_i8_dequantize: ")


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=1 << 30), dict(n=-1), dict(n=1 << 30), dict(k=0), dict(k=-1), dict(k=131072, xs=0, cs=0),
    dict(yt=E4M3), dict(yt=I8), dict(yt=-1), dict(mode=NONE), dict(mode=3), dict(xs=127), dict(cs=127), dict(ys=7),
    dict(xs=1 << 30), dict(x=None), dict(xsc=None), dict(codes=None), dict(scales=None), dict(y=None), dict(xsc=Q + 2),
    dict(scales=S + 1), dict(bias=V + 2), dict(y=T + 1), dict(yt=F32, y=T + 2), dict(y=P), dict(y=R)])
def test_i8_linear_refuses(kw):
    assert linear(**kw) == fx.FX_INVALID_ARGUMENT
    assert fx.lib().fx_last_error().startswith(b"fx_i8_linear: ")


def test_no_rows_is_no_error():
    assert norm(rows=0, x=None, y=None) == fx.FX_OK
    assert backward(rows=0, dy=None, h=None, mean=None, rstd=None, dx=None) == fx.FX_OK
    assert linear(rows=0, x=None, y=None) == fx.FX_OK
    assert linear(n=0, codes=None, scales=None, y=None) == fx.FX_OK
    assert quantize(rows=0, x=None, codes=None, scales=None) == fx.FX_OK
    assert dequantize(rows=0, y=None, codes=None, scales=None) == fx.FX_OK


def test_other_operators_take_no_i8():
    L = fx.lib()
    assert L.fx_rms_norm(P, BF16, 4, 64, 64, None, BF16, 64, None, 64, None, BF16, 1e-6, Q, I8, 64, R, ROW, None) == fx.FX_INVALID_ARGUMENT
    assert L.fx_w4_linear(P, I8, 4, 128, Q, ROW, R, S, F16, None, 8, 128, 32, None, T, BF16, 8, None) == fx.FX_INVALID_ARGUMENT


def test_python_names_of_types_and_modes():
    with pytest.raises(KeyError):
        fx.layer_norm_dev(P, Q, 1, 8, x_type="f64")
    with pytest.raises(KeyError):
        fx.i8_linear_dev(P, Q, 1, 8, 32, R, S, T, x_scale_mode="column")
    with pytest.raises(fx.FxError) as e:
        fx.i8_linear_dev(P, Q, 1, 8, 131072, R, S, T)
    assert e.value.code == fx.FX_INVALID_ARGUMENT and "131071" in str(e.value)
