"""The layer norm and its backward pass on the GPU against plain implementations in 64 bits.

Tolerances count roundings; u = 2^-24 is half a step of f32, HALF[t] half a step of type t, both relative. A row's sum is made
of at most 64 additions in a row per thread and a tree of at most 15 levels: its error is below 80 u times the sum of
magnitudes.

Forward, with t = h - mean in units of the standard deviation, z = t r:
- with a residual h is rounded once (u |h|), t once more (u |t|), and the mean's correction, a sum of the t, is off by 82 u of their mean
  magnitude, which is below 1 in those units; the rounding of h moves the mean by as much as it moves h: 2 u max|h| r in all.
- the variance is off by 84 u relative, and by 2 u max|h| r (the h it is made of); its root by half of both; the hardware's
  reciprocal root adds 4 u, the products two: |z| (50 u + u max|h| r).
- the first mean is off by 80 u of the row's size, |h| r = far: the t are that much larger than the z, at most k = 1 + 80 u far
  times, and so are their errors; the variance takes the square of that off again.
- weight and bias: a rounding each, relative to |z w| and to the result.
Backward, g = dy weight, s1 = mean(g), s2 = mean(g z): s1 is off by 82 u mean|g|, s2 by 87 u mean|g z| (z itself by 3 u), and
each remaining operation by u of its size; all times rstd. Sums over rows: a thread adds at most max(8, rows / 148 + 1) rows one
after the other, shuffles 5, warps 4, and lines of the workspace in eight lots of at most 148 and then 8; each addition is off by
u of the sum of magnitudes, each product by 5 u."""
import itertools

import pytest

import fenix_b200 as fx
from test_token_gpu import HALF, TINY, U, check_close, ptr, rows_of, stream, tt

pytestmark = pytest.mark.gpu

TOP = {"e4m3": 448.0, "i8": 127.0}


def dtype(torch, name):
    return torch.int8 if name == "i8" else tt(torch, name)


# ---- forward ----------------------------------------------------------------------------------------------------


def norm_want(torch, x, residual, weight, bias, eps):
    """(h, mean, rstd, v, tolerance of v) in f64."""
    h = x.double()
    if residual is not None:
        h = h + residual.double()
    var, mean = torch.var_mean(h, 1, correction=0, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    z = (h - mean) * r
    far = h.abs().amax(1, keepdim=True) * r
    k, far = 1 + 80 * U * far, far if residual is not None else 0.0
    w = weight.double() if weight is not None else torch.ones_like(z[0])
    v = z * w
    tol = U * w.abs() * (3 * far + 84 * k + z.abs() * (52 * k * k + far)) + U * v.abs()
    if bias is not None:
        v = v + bias.double()
    return h, mean[:, 0], r[:, 0], v, tol + U * v.abs()


def within(got, want, tol):
    over = ((got.double() - want).abs() - tol).max().item()
    assert over <= 0, (over, (got.double() - want).abs().max().item())


def check_norm(torch, x, residual, weight, bias, eps, yt, y, scale, mode):
    h, mean, r, v, tol = norm_want(torch, x, residual, weight, bias, eps)
    if mode is None:
        within(y, v, tol + HALF[yt] * (v.abs() + tol) + TINY[yt])
        return
    top = TOP[yt]
    if mode == "row":
        within(scale, v.abs().amax(1).clamp(min=1e-30) / top, tol.amax(1) / top + 4 * U * scale.double())
        s = scale.double()[:, None]
    else:
        s = scale.double()
    lim = (v / s).clamp(-top, top)
    rel = tol / s + 4 * U * lim.abs()
    within(y.float(), lim, rel + 0.5 * (1 + 4 * U) if yt == "i8" else HALF["e4m3"] * (lim.abs() + rel) + rel + TINY["e4m3"] / 2)


def run_norm(torch, rows, cols, xt="bf16", yt="bf16", rt="bf16", wt="bf16", mode=None, residual=True, keep_sum=True,
             weight=True, bias=True, stats=True, strides=(0, 0, 0, 0), offset=0, seed=0, eps=1e-5, spread=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    xs, rs, ss, ys = strides
    _, x = rows_of(torch, rows, cols, tt(torch, xt), xs, offset)
    x.copy_(torch.randn(rows, cols, generator=g, device="cuda") * spread + shift)
    r = s = w = b = scale = mean = rstd = None
    if residual:
        _, r = rows_of(torch, rows, cols, tt(torch, rt), rs, offset)
        r.copy_(torch.randn(rows, cols, generator=g, device="cuda") * 2)
    if keep_sum:
        sbuf, s = rows_of(torch, rows, cols, tt(torch, rt), ss, offset, 7.0)
    if weight:
        w = (torch.rand(cols + offset, generator=g, device="cuda") + 0.5).to(tt(torch, wt))[offset:]
    if bias:
        b = torch.randn(cols + offset, generator=g, device="cuda").to(tt(torch, wt))[offset:]
    if stats:
        mean, rstd = torch.full((rows + 1,), 5.0, device="cuda"), torch.full((rows + 1,), 5.0, device="cuda")
    ybuf, y = rows_of(torch, rows, cols, dtype(torch, yt), ys, offset, 7)
    if mode == "row":
        scale = torch.full((rows + 1,), 5.0, device="cuda")
    elif mode == "tensor":
        scale = torch.tensor([3.0 / TOP[yt]], device="cuda")
    fx.layer_norm_dev(ptr(x), ptr(y), rows, cols, xt, yt, ptr(w), ptr(b), wt, eps, xs, ys, ptr(r), rt, rs, ptr(s), ss, ptr(mean),
                      ptr(rstd), ptr(scale), mode, stream(torch))
    torch.cuda.synchronize()
    h, m, rs_, v, tol = norm_want(torch, x, r, w, b, eps)
    if keep_sum:
        check_close(torch, s, h, HALF[rt] + 2 * U, TINY[rt])
        s.fill_(7.0)
        assert bool((sbuf == 7.0).all())  # nothing outside the rows was written
    if stats:
        top = h.abs().amax(1)
        within(mean[:rows], m, U * (3 * top + 84 / rs_))
        within(rstd[:rows], rs_, rs_ * U * (50 * (1 + 80 * U * top * rs_) ** 2 + top * rs_))
        assert mean[rows].item() == 5.0 and rstd[rows].item() == 5.0
    if mode == "row":
        assert scale[rows].item() == 5.0
        scale = scale[:rows]
    check_norm(torch, x, r, w, b, eps, yt, y, scale, mode)
    y.copy_(torch.full((rows, cols), 7.0, device="cuda"))
    assert bool((ybuf.float() == 7.0).all())


@pytest.mark.parametrize("cols", [1, 2, 7, 8, 31, 32, 64, 72, 100, 128, 136, 255, 256, 264, 320, 328, 512, 520, 1000, 1024, 1032, 2048,
                                  2049, 4096, 4104, 5119, 5120, 6144, 7168, 8192, 8200, 10000, 16384, 16392, 32760, 32767, 32768])
@pytest.mark.parametrize("rows", [1, 3, 300])
def test_norm_extents(cuda_torch, rows, cols):
    run_norm(cuda_torch, rows, cols, yt="i8", mode="row", seed=cols)
    run_norm(cuda_torch, rows, cols, yt="bf16", residual=False, keep_sum=False, seed=cols + 1)


@pytest.mark.parametrize("cols", [24, 64, 120, 128, 248, 256, 312, 320, 504, 512, 1016, 1024, 2040, 2048, 4096, 5112, 6136, 8184, 16384])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_teams_that_walk(cuda_torch, cols, residual):
    """Enough rows that blocks stay and take several, the last of them with teams that have none left."""
    rows = max(2400, 10_000_000 // cols) + 3
    run_norm(cuda_torch, rows, cols, "f16" if cols % 3 else "bf16", "e4m3", mode="row", residual=residual, keep_sum=residual, seed=cols)
    run_norm(cuda_torch, rows, cols, "bf16", "bf16", residual=residual, keep_sum=residual, seed=cols)
    if not residual:  # h is x, and is stored all the same, in any type
        for rt in ("f32", "f16", "bf16"):
            run_norm(cuda_torch, rows, cols, "bf16", "i8", rt, "bf16", "row", residual=False, keep_sum=True, seed=cols)
            run_norm(cuda_torch, rows, cols, "f16", "f32", rt, "f32", residual=False, keep_sum=True, bias=False, seed=cols)


@pytest.mark.parametrize("xt,yt,rt", list(itertools.product(["f32", "f16", "bf16"], ["f32", "f16", "bf16", "e4m3", "i8"],
                                                        ["f32", "f16", "bf16"])))
def test_norm_types(cuda_torch, xt, yt, rt):
    wt = {"f32": "f16", "f16": "bf16", "bf16": "f32"}[xt]
    for cols in (328, 333, 2048):
        for mode in ("row", "tensor") if yt in TOP else (None,):
            run_norm(cuda_torch, 37, cols, xt, yt, rt, wt, mode, seed=cols)


@pytest.mark.parametrize("residual,keep_sum,weight,bias,stats", list(itertools.product([False, True], repeat=5)))
def test_norm_optional_operands(cuda_torch, residual, keep_sum, weight, bias, stats):
    for cols in (96, 4096, 4097):
        run_norm(cuda_torch, 5, cols, "f16", "f32", "f32", "f32", None, residual, keep_sum, weight, bias, stats)


@pytest.mark.parametrize("offset", [0, 1, 3, 8])
@pytest.mark.parametrize("strides", [(0, 0, 0, 0), (528, 520, 544, 536), (521, 0, 0, 0), (0, 523, 0, 0), (0, 0, 525, 0),
                                     (0, 0, 0, 527)])
def test_norm_strides_and_offsets(cuda_torch, strides, offset):
    for yt, mode in (("e4m3", "row"), ("i8", "tensor"), ("f16", None)):
        run_norm(cuda_torch, 9, 512, "bf16", yt, "f32", mode=mode, strides=strides, offset=offset)


@pytest.mark.parametrize("shift", [1e3, -1e5, 3e7])
def test_norm_rows_far_from_zero(cuda_torch, shift):
    """The variance of f32 rows far from zero is that of what is left of them: sums of squares would lose it."""
    for rows, cols in ((4, 100), (4, 4096), (300, 64), (200, 5119)):
        run_norm(cuda_torch, rows, cols, "f32", "f32", "f32", "f32", residual=False, keep_sum=False, shift=shift, spread=100.0)
    for rows, cols in ((20000, 64), (3000, 4096)):
        run_norm(cuda_torch, rows, cols, "bf16", "f32", "bf16", "f32", residual=False, keep_sum=False, shift=shift / 1e3, spread=10.0)


def test_norm_rows_past_32_bits(cuda_torch):
    torch = cuda_torch
    rows, cols, stride = 1100, 256, 1 << 22
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    run_norm(torch, rows, cols, strides=(stride, 0, stride, 0))
    torch.cuda.empty_cache()
    run_norm(torch, rows, cols, residual=False, keep_sum=False, yt="i8", mode="row", strides=(0, 0, 0, stride))
    torch.cuda.empty_cache()


def test_norm_many_rows(cuda_torch):
    run_norm(cuda_torch, 70001, 48, yt="e4m3", mode="row")
    run_norm(cuda_torch, 200001, 8, "f16", "f16", "f16")
    run_norm(cuda_torch, 200001, 9, "f32", "i8", "f16", mode="row")


def test_norm_in_place(cuda_torch):
    torch = cuda_torch
    for rows, cols in ((11, 40), (11, 77), (11, 4096), (11, 20000), (30000, 64), (4000, 4096)):
        x = torch.randn(rows, cols, device="cuda").bfloat16()
        r = torch.randn(rows, cols, device="cuda").bfloat16()
        h, _, _, v, tol = norm_want(torch, x, r, None, None, 1e-5)
        x1, r1 = x.clone(), r.clone()  # the sum in place of the residual, the result in place of x
        fx.layer_norm_dev(ptr(x1), ptr(x1), rows, cols, residual_ptr=ptr(r1), sum_ptr=ptr(r1), stream=stream(torch))
        within(x1, v, tol + HALF["bf16"] * (v.abs() + tol))
        check_close(torch, r1, h, HALF["bf16"] + 2 * U, TINY["bf16"])
        x2, y2 = x.clone(), torch.empty_like(x)  # the sum in place of x
        fx.layer_norm_dev(ptr(x2), ptr(y2), rows, cols, residual_ptr=ptr(r), sum_ptr=ptr(x2), stream=stream(torch))
        assert torch.equal(x2, r1) and torch.equal(y2, x1)


@pytest.mark.parametrize("rows,cols", [(12, 64), (12, 100), (12, 4000), (12, 9000), (3000, 64), (9000, 320), (3000, 1000), (1600, 4096)])
def test_norm_extreme_rows(cuda_torch, rows, cols):
    torch = cuda_torch
    inf, nan = float("inf"), float("nan")
    for xt in ("f32", "bf16"):
        g = torch.Generator(device="cuda").manual_seed(cols)
        x = torch.randn(rows, cols, generator=g, device="cuda")
        x[1] = 0.0
        x[2, 5], x[3, 6], x[7, cols - 1] = inf, nan, -inf
        x[4] *= 1e-22   # squares below f32's range: eps alone is left
        x[5] *= 1e25    # squares past f32's range
        x[6] *= 4e37
        x[8] = 0.25     # all alike
        x[9] = 3.0e38   # the same, and their sum past f32's range
        x = x.to(tt(torch, xt))
        gain = torch.ones(cols, device="cuda")
        shift = torch.full((cols,), 0.5, device="cuda")
        fine = [i for i in range(rows) if i not in (2, 3, 7, 9)]
        for yt, mode in (("f32", None), ("bf16", None), ("e4m3", "row"), ("e4m3", "tensor"), ("i8", "row"), ("i8", "tensor")):
            y = torch.empty(rows, cols, dtype=dtype(torch, yt), device="cuda")
            scale = torch.full((rows if mode == "row" else 1,), 0.02, device="cuda") if mode else None
            mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
            fx.layer_norm_dev(ptr(x), ptr(y), rows, cols, xt, yt, ptr(gain), ptr(shift), "f32", 1e-6, mean_ptr=ptr(mean),
                              rstd_ptr=ptr(rstd), scale_ptr=ptr(scale), scale_mode=mode, stream=stream(torch))
            torch.cuda.synchronize()
            got = y.float()
            check_norm(torch, x[fine], None, gain, shift, 1e-6, yt, y[fine], scale[fine] if mode == "row" else scale, mode)
            assert bool(rstd[[2, 3, 7]].isnan().all()) and not bool(mean[[2, 3, 7]].isfinite().any())
            assert bool(rstd[fine].isfinite().all()) and bool(got[9].isfinite().all())
            if yt == "i8":
                assert bool((y[[2, 3, 7]] == 0).all()) and (mode == "tensor" or bool(scale[[2, 3, 7]].isnan().all()))
            else:
                assert bool(got[[2, 3, 7]].isnan().all()) and (mode != "row" or bool(scale[[2, 3, 7]].isnan().all()))


@pytest.mark.parametrize("scale", [1e-40, 3e38])
@pytest.mark.parametrize("yt", ["e4m3", "i8"])
def test_norm_tensor_scales_at_the_ends(cuda_torch, yt, scale):
    torch = cuda_torch
    x = torch.randn(6, 200, device="cuda")
    x[2] = 1.0
    y = torch.empty(6, 200, dtype=dtype(torch, yt), device="cuda")
    s = torch.tensor([scale], device="cuda")
    fx.layer_norm_dev(ptr(x), ptr(y), 6, 200, "f32", yt, scale_ptr=ptr(s), scale_mode="tensor", stream=stream(torch))
    torch.cuda.synchronize()
    got = y.float()
    assert bool((got[2] == 0).all())
    assert bool((got[0].abs() == (TOP[yt] if scale < 1 else 0.0)).all())


# ---- backward ---------------------------------------------------------------------------------------------------


def backward_want(torch, dy, h, mean, rstd, weight, dsum):
    """(dx, its tolerance before it is rounded, dweight, dbias, sums of magnitudes of both) in f64."""
    dy, m, r = dy.double(), mean.double()[:, None], rstd.double()[:, None]
    z = (h.double() - m) * r
    g = dy * weight.double() if weight is not None else dy
    s1, s2 = g.mean(1, keepdim=True), (g * z).mean(1, keepdim=True)
    dx = (g - s1 - z * s2) * r
    tol = U * r.abs() * (88 * g.abs().mean(1, keepdim=True) + 92 * z.abs() * (g * z).abs().mean(1, keepdim=True) +
                         8 * (g.abs() + (z * s2).abs() + s1.abs()))
    if dsum is not None:
        dx = dx + dsum.double()
    return dx, tol + U * dx.abs(), (dy * z).sum(0), dy.sum(0), (dy * z).abs().sum(0), dy.abs().sum(0)


def run_backward(torch, rows, cols, dyt="bf16", ht="bf16", wt="bf16", dxt="bf16", weight=True, dsum=True, dx=True, sums="wb",
                 accumulate=False, strides=(0, 0, 0, 0), offset=0, seed=0, in_place=None):
    g = torch.Generator(device="cuda").manual_seed(seed + cols)
    ds, hs, ss, xs = strides
    rand = lambda: torch.randn(rows, cols, generator=g, device="cuda")  # noqa: E731
    _, dy = rows_of(torch, rows, cols, tt(torch, dyt), ds, offset)
    _, h = rows_of(torch, rows, cols, tt(torch, ht), hs, offset)
    dy.copy_(rand())
    h.copy_(rand() * 3 + torch.randn(rows, 1, generator=g, device="cuda"))
    var, mean = torch.var_mean(h.double(), 1, correction=0)
    mean, rstd = mean.float(), (1 / torch.sqrt(var + 1e-5)).float()
    w = d = out = dw = db = work = xbuf = None
    if weight:
        w = (torch.rand(cols + offset, generator=g, device="cuda") + 0.5).to(tt(torch, wt))[offset:]
    if dsum:
        _, d = rows_of(torch, rows, cols, tt(torch, dxt), ss, offset)
        d.copy_(rand())
    want, tol, ww, wb, aw, ab = backward_want(torch, dy, h, mean, rstd, w, d)
    if in_place:
        out = {"dy": dy, "h": h, "dsum": d}[in_place]
    elif dx:
        xbuf, out = rows_of(torch, rows, cols, tt(torch, dxt), xs, offset, 7.0)
    start = torch.randn(2, cols, generator=g, device="cuda")
    if "w" in sums:
        dw = torch.cat((start[0], start[0, :1]))
    if "b" in sums:
        db = torch.cat((start[1], start[1, :1]))
    if sums:
        size = fx.layer_norm_backward_workspace(rows, cols)
        work = torch.full((size + 16,), 0xa5, dtype=torch.uint8, device="cuda")
    fx.layer_norm_backward_dev(ptr(dy), ptr(h), ptr(mean), ptr(rstd), rows, cols, dyt, ht, ptr(w), wt, ptr(d), ptr(out), dxt,
                               ptr(dw), ptr(db), accumulate, ptr(work), size if sums else 0, ds, hs, ss, xs, stream(torch))
    torch.cuda.synchronize()
    if out is not None:
        within(out, want, tol + HALF[dxt] * (want.abs() + tol) + TINY[dxt])
    if xbuf is not None:
        out.fill_(7.0)
        assert bool((xbuf == 7.0).all())
    adds = max(8, rows // 148 + 1) + 5 + 4 + 148 + 8 + 1
    for got, full, mag, first in ((dw, ww, aw, start[0].double()), (db, wb, ab, start[1].double())):
        if got is None:
            continue
        if accumulate:
            full, mag = full + first, mag + first.abs()
        within(got[:cols], full, U * (adds + 5) * mag)
        assert got[cols].item() == first[0].item()
    if sums:
        assert bool((work[size:] == 0xa5).all())


@pytest.mark.parametrize("cols", [1, 2, 7, 8, 31, 32, 64, 65, 72, 100, 128, 255, 256, 264, 320, 511, 512, 520, 1000, 1024, 1032, 2048, 2049,
                                  4095, 4096, 4104, 5119, 5120, 6144, 6150, 7168, 8191, 8192, 8193, 8200, 10000, 16384, 32767, 32768])
@pytest.mark.parametrize("rows", [1, 3, 300])
def test_backward_extents(cuda_torch, rows, cols):
    run_backward(cuda_torch, rows, cols)
    run_backward(cuda_torch, rows, cols, "f32", "f32", "f32", "f32", dsum=False)


@pytest.mark.parametrize("cols", [24, 64, 120, 128, 248, 256, 312, 320, 504, 512, 1016, 1024, 2040, 2048, 4096, 5112, 6136, 8184, 9000, 16384])
def test_backward_many_rows(cuda_torch, cols):
    rows = max(2400, 10_000_000 // cols) + 3
    run_backward(cuda_torch, rows, cols, "f16", "bf16", "f32", "bf16")
    run_backward(cuda_torch, rows, cols, "bf16", "bf16", "bf16", "bf16", dsum=False, accumulate=True)
    run_backward(cuda_torch, rows // 2, cols - 1, "f16", "f16", "f16", "f16", dsum=False)


@pytest.mark.parametrize("dyt,ht,dxt", list(itertools.product(["f32", "f16", "bf16"], repeat=3)))
def test_backward_types(cuda_torch, dyt, ht, dxt):
    wt = {"f32": "f16", "f16": "bf16", "bf16": "f32"}[ht]
    for cols in (328, 333, 2048, 8448):
        run_backward(cuda_torch, 37, cols, dyt, ht, wt, dxt)


@pytest.mark.parametrize("weight,dsum,dx,sums", [c for c in itertools.product([False, True], [False, True], [False, True],
                                                                           ["", "w", "b", "wb"]) if c[2] or c[3]])
def test_backward_optional_operands(cuda_torch, weight, dsum, dx, sums):
    for rows, cols in ((5, 96), (400, 1024), (50, 4097), (40, 9000)):
        run_backward(cuda_torch, rows, cols, weight=weight, dsum=dsum, dx=dx, sums=sums, accumulate=sums == "w")


@pytest.mark.parametrize("offset", [0, 1, 3, 8])
@pytest.mark.parametrize("strides", [(0, 0, 0, 0), (528, 520, 544, 536), (521, 0, 0, 0), (0, 523, 0, 0), (0, 0, 525, 0),
                                     (0, 0, 0, 527)])
def test_backward_strides_and_offsets(cuda_torch, strides, offset):
    run_backward(cuda_torch, 9, 512, strides=strides, offset=offset)
    run_backward(cuda_torch, 9, 512, "f32", "bf16", "f16", "f32", strides=strides, offset=offset)


@pytest.mark.parametrize("where", ["dy", "h", "dsum"])
def test_backward_in_place(cuda_torch, where):
    for rows, cols in ((11, 40), (11, 77), (700, 4096), (60, 9001), (20000, 64), (300, 9008), (300, 16384), (200, 20000)):
        run_backward(cuda_torch, rows, cols, in_place=where)
        run_backward(cuda_torch, rows, cols, "f32", "f32", "f32", "f32", in_place=where)


def test_backward_past_32_bits(cuda_torch):
    torch = cuda_torch
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free device memory")
    stride = 1 << 22
    for strides in ((stride, 0, 0, 0), (0, stride, 0, 0), (0, 0, stride, 0), (0, 0, 0, stride)):
        run_backward(torch, 1100, 256, strides=strides)
        torch.cuda.empty_cache()
    run_backward(torch, 1100, 8704, strides=(stride, 0, 0, 0))
    torch.cuda.empty_cache()


def test_backward_without_rows(cuda_torch):
    torch = cuda_torch
    dw, db = torch.ones(64, device="cuda"), torch.ones(64, device="cuda")
    fx.layer_norm_backward_dev(0, 0, 0, 0, 0, 64, dweight_ptr=ptr(dw), dbias_ptr=ptr(db), accumulate=True, stream=stream(torch))
    assert bool((dw == 1).all()) and bool((db == 1).all())
    fx.layer_norm_backward_dev(0, 0, 0, 0, 0, 64, dweight_ptr=ptr(dw), dbias_ptr=ptr(db), stream=stream(torch))
    torch.cuda.synchronize()
    assert bool((dw == 0).all()) and bool((db == 0).all())


def test_backward_rows_not_finite_stay_apart(cuda_torch):
    torch = cuda_torch
    for rows, cols in ((6, 100), (3000, 64), (600, 4096), (6, 9000)):
        h, dy = torch.randn(rows, cols, device="cuda"), torch.randn(rows, cols, device="cuda")
        mean, rstd = h.mean(1), 1 / h.std(1, correction=0)
        dx = torch.empty_like(h)
        h[2, 5], dy[3, 6] = float("nan"), float("inf")
        fx.layer_norm_backward_dev(ptr(dy), ptr(h), ptr(mean), ptr(rstd), rows, cols, "f32", "f32", dx_ptr=ptr(dx), dx_type="f32",
                                   stream=stream(torch))
        torch.cuda.synchronize()
        keep = [i for i in range(rows) if i not in (2, 3)]
        assert bool(dx[keep].isfinite().all()) and bool(dx[2].isnan().all()) and not bool(dx[3].isfinite().any())


def test_backward_is_the_formulas_gradient(cuda_torch):
    """From fx_layer_norm's own statistics, against the formula differentiated by torch in 64 bits and against differences."""
    torch = cuda_torch
    rows, cols = 5, 24
    g = torch.Generator(device="cuda").manual_seed(3)
    x, r, dv, ds = (torch.randn(rows, cols, generator=g, device="cuda") for _ in range(4))
    w, b = torch.rand(cols, generator=g, device="cuda") + 0.5, torch.randn(cols, generator=g, device="cuda")
    y, s, dx = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    mean, rstd, dw, db = (torch.empty(n, device="cuda") for n in (rows, rows, cols, cols))
    work = torch.empty(fx.layer_norm_backward_workspace(rows, cols), dtype=torch.uint8, device="cuda")
    fx.layer_norm_dev(ptr(x), ptr(y), rows, cols, "f32", "f32", ptr(w), ptr(b), "f32", 1e-5, residual_ptr=ptr(r), residual_type="f32",
                      sum_ptr=ptr(s), mean_ptr=ptr(mean), rstd_ptr=ptr(rstd), stream=stream(torch))
    fx.layer_norm_backward_dev(ptr(dv), ptr(s), ptr(mean), ptr(rstd), rows, cols, "f32", "f32", ptr(w), "f32", ptr(ds), ptr(dx),
                               "f32", ptr(dw), ptr(db), False, ptr(work), work.numel(), stream=stream(torch))
    torch.cuda.synchronize()

    def loss(h, w, b):
        var, m = torch.var_mean(h, 1, correction=0, keepdim=True)
        return (((h - m) / torch.sqrt(var + 1e-5) * w + b) * dv.double()).sum() + (h * ds.double()).sum()

    args = [t.double().requires_grad_() for t in (x.double() + r.double(), w, b)]
    loss(*args).backward()
    # the sums here are of 24 values of some units: 100 u of them covers the counts above
    for got, a in zip((dx, dw, db), args):
        within(got, a.grad, 100 * U * 24 * torch.ones_like(a.grad) * 4)
    with torch.no_grad():
        for got, i in ((dx, 0), (dw, 1), (db, 2)):
            flat = args[i].detach().clone().reshape(-1)
            for at in range(0, flat.numel(), 7):
                ends = []
                for step in (1e-5, -1e-5):
                    moved = flat.clone()
                    moved[at] += step
                    ends.append(loss(*[moved.view_as(args[i]) if j == i else args[j] for j in range(3)]))
                # a central difference of step 1e-5 is off by some 1e-10 times the third derivative and 1e-16 / 1e-5 of the loss
                assert abs((ends[0] - ends[1]).item() / 2e-5 - got.reshape(-1)[at].item()) < 1e-3


def test_forward_and_backward_captured_side_by_side(cuda_torch):
    """A training step's norm, forward and back, in two graphs on two streams with a workspace each, and eagerly beside them;
    every repetition gives the same bits."""
    torch = cuda_torch

    class Step:
        def __init__(self, rows, cols, seed):
            g = torch.Generator(device="cuda").manual_seed(seed)
            e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
            self.rows, self.cols = rows, cols
            self.x, self.r, self.dy, self.ds = (torch.randn(rows, cols, generator=g, device="cuda").bfloat16() for _ in range(4))
            self.w, self.b = (torch.rand(cols, generator=g, device="cuda").bfloat16() for _ in range(2))
            self.y, self.s, self.dx = e(rows, cols), e(rows, cols), e(rows, cols)
            f = torch.float32
            self.mean, self.rstd, self.dw, self.db = e(rows, dtype=f), e(rows, dtype=f), e(cols, dtype=f), e(cols, dtype=f)
            self.work = e(fx.layer_norm_backward_workspace(rows, cols), dtype=torch.uint8)

        def run(self):
            st = stream(torch)
            fx.layer_norm_dev(ptr(self.x), ptr(self.y), self.rows, self.cols, weight_ptr=ptr(self.w), bias_ptr=ptr(self.b),
                              residual_ptr=ptr(self.r), sum_ptr=ptr(self.s), mean_ptr=ptr(self.mean), rstd_ptr=ptr(self.rstd), stream=st)
            fx.layer_norm_backward_dev(ptr(self.dy), ptr(self.s), ptr(self.mean), ptr(self.rstd), self.rows, self.cols,
                                       weight_ptr=ptr(self.w), dsum_ptr=ptr(self.ds), dx_ptr=ptr(self.dx), dweight_ptr=ptr(self.dw),
                                       dbias_ptr=ptr(self.db), work_ptr=ptr(self.work), work_bytes=self.work.numel(), stream=st)

        def outputs(self):
            return [t.clone() for t in (self.y, self.s, self.dx, self.dw, self.db, self.mean, self.rstd)]

    for rows, cols in ((700, 1024), (5000, 320), (60, 9000), (3, 4096)):
        steps = [Step(rows, cols, i) for i in range(3)]
        first = []
        for st in steps:
            st.run()
            torch.cuda.synchronize()
            first.append(st.outputs())
            want, tol, ww, wb, aw, ab = backward_want(torch, st.dy, st.s, st.mean, st.rstd, st.w, st.ds)
            within(st.dx, want, tol + HALF["bf16"] * (want.abs() + tol) + TINY["bf16"])
        streams = [torch.cuda.Stream() for _ in steps]
        graphs = []
        for st, on in zip(steps[:2], streams):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=on):
                st.run()
            graphs.append(g)
        for _ in range(4):
            for g, on in zip(graphs, streams):
                with torch.cuda.stream(on):
                    g.replay()
            with torch.cuda.stream(streams[2]):
                steps[2].run()
        torch.cuda.synchronize()
        for st, was in zip(steps, first):
            assert all(torch.equal(p, q) for p, q in zip(st.outputs(), was))


@pytest.mark.parametrize("rows,cols", [(40, 256), (700, 1024), (3000, 4096), (500, 9000), (60, 1001)])
def test_one_workspace_call_after_call(cuda_torch, rows, cols):
    """Calls that follow one another on a stream share a workspace, an input that each call overwrites, and accumulated sums."""
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(cols)
    xs = [torch.randn(rows, cols, generator=g, device="cuda").bfloat16() * (i + 1) for i in range(12)]
    work = torch.empty(fx.layer_norm_backward_workspace(rows, cols), dtype=torch.uint8, device="cuda")
    s, y, dx = torch.empty_like(xs[0]), torch.empty_like(xs[0]), torch.empty_like(xs[0])
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    total = torch.zeros(2, cols, device="cuda")

    def run(x, dw, db, accumulate, together):
        st = stream(torch)
        fx.layer_norm_dev(ptr(x), ptr(y), rows, cols, residual_ptr=ptr(x), sum_ptr=ptr(s), mean_ptr=ptr(mean), rstd_ptr=ptr(rstd), stream=st)
        if not together:
            torch.cuda.synchronize()
        fx.layer_norm_backward_dev(ptr(y), ptr(s), ptr(mean), ptr(rstd), rows, cols, dx_ptr=ptr(dx), dweight_ptr=ptr(dw), dbias_ptr=ptr(db),
                                   accumulate=accumulate, work_ptr=ptr(work), work_bytes=work.numel(), stream=st)
        if not together:
            torch.cuda.synchronize()

    apart = [torch.empty(2, cols, device="cuda") for _ in xs]
    for x, out in zip(xs, apart):
        run(x, out[0], out[1], False, False)
    for _ in range(5):
        close = [torch.empty(2, cols, device="cuda") for _ in xs]
        total.zero_()
        torch.cuda.synchronize()
        for x, out in zip(xs, close):
            run(x, out[0], out[1], False, True)
            run(x, total[0], total[1], True, True)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(apart, close))
        want = torch.zeros_like(total)
        for out in apart:
            want += out
        assert torch.equal(total, want)
