"""The token-row operators on the GPU against plain implementations in 64 bits.

Tolerances count roundings. u = 2^-24 is half a step of f32, HALF[t] half a step of type t, both relative.
- rms_norm: a row's sum of squares is made of at most 64 additions in a row per thread and a tree of at most 15
  levels, so its relative error is below 80 u and its square root's below 40 u; the hardware's reciprocal square
  root adds 4 u, the sum h, the two products and the quotient by the scale one or two each: 48 u in all.
- w4_linear: a weight may be rounded once to x's 16-bit type (f16 for e4m3), an error below HALF[t] |w| whose
  sign follows the input's, so that the error of a sum over symmetric random inputs exceeds
  4 HALF[t] sqrt(sum (w x)^2) with probability below 2 exp(-8) per output times the share of outputs with errors at
  their bounds; errors are spread over the step (variance a third of the bound's square), so 4 is 6.9 standard
  deviations. The f32 sums add at most (k / 16) 2^-22 sum |w x|. The result is rounded once more to y's type.
- Inputs that are whole numbers times powers of two leave nothing to round: those results are exact, and
  whatever a kernel reads or writes in the wrong place shows.
"""
import itertools

import pytest

import fenix_b200 as fx

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8, "e4m3": 2.0 ** -4}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133, "e4m3": 2.0 ** -9}  # smallest subnormal
NORM_TOL = 48 * U


def tt(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}[name]


def ptr(t):
    return None if t is None else t.data_ptr()


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


def rows_of(torch, rows, cols, dtype, stride=0, offset=0, fill=None):
    """A [rows][cols] view with `stride` elements a row, `offset` elements into its allocation."""
    stride = stride or cols
    buf = torch.empty(offset + rows * stride + 16, dtype=dtype, device="cuda")
    if fill is not None:
        buf.fill_(fill)
    return buf, buf.as_strided((rows, cols), (stride, 1), offset)


# ---- rms_norm ---------------------------------------------------------------------------------------------------


def norm_want(torch, x, residual, weight, eps):
    h = x.double()
    if residual is not None:
        h = h + residual.double()
    v = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    return h, v * weight.double() if weight is not None else v


def check_close(torch, got, want, rel, tiny):
    err = (got.double() - want).abs()
    over = (err - (rel * want.abs() + tiny)).max().item()
    assert over <= 0, (over, err.max().item())


def run_norm(torch, rows, cols, xt="bf16", yt="bf16", rt="bf16", wt="bf16", mode=None, residual=True, keep_sum=True,
             weight=True, strides=(0, 0, 0, 0), offset=0, seed=0, eps=1e-5, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    xs, rs, ss, ys = strides
    _, x = rows_of(torch, rows, cols, tt(torch, xt), xs, offset)
    x.copy_(torch.randn(rows, cols, generator=g, device="cuda") * spread)
    r = s = w = scale = None
    if residual:
        _, r = rows_of(torch, rows, cols, tt(torch, rt), rs, offset)
        r.copy_(torch.randn(rows, cols, generator=g, device="cuda") * 2)
    if keep_sum:
        sbuf, s = rows_of(torch, rows, cols, tt(torch, rt), ss, offset, 7.0)
    if weight:
        w = (torch.rand(cols + offset, generator=g, device="cuda") + 0.5).to(tt(torch, wt))[offset:]
    ybuf, y = rows_of(torch, rows, cols, tt(torch, yt), ys, offset, 7.0)
    if mode == "row":
        scale = torch.full((rows + 1,), 5.0, device="cuda")
    elif mode == "tensor":
        scale = torch.tensor([0.0125], device="cuda")
    fx.rms_norm_dev(ptr(x), ptr(y), rows, cols, xt, yt, ptr(w), wt, eps, xs, ys, ptr(r), rt, rs, ptr(s), ss, ptr(scale),
                    mode, stream(torch))
    torch.cuda.synchronize()
    h, v = norm_want(torch, x, r, w, eps)
    if keep_sum:
        check_close(torch, s, h, HALF[rt] + 2 * U, TINY[rt])
        sbuf.as_strided((rows, cols), (ss or cols, 1), offset).fill_(7.0)
        assert bool((sbuf == 7.0).all())  # nothing outside the rows was written
    if mode is None:
        check_close(torch, y, v, HALF[yt] + NORM_TOL, TINY[yt])
    else:
        if mode == "row":
            want = v.abs().amax(1).clamp(min=1e-30) / 448
            check_close(torch, scale[:rows], want, NORM_TOL, 0.0)
            assert scale[rows].item() == 5.0
            scale = scale[:rows, None]
        q = y.double()
        lim = (v / scale.double()).clamp(-448, 448)
        check_close(torch, q, lim, HALF["e4m3"] + NORM_TOL, TINY["e4m3"] / 2 * (1 + NORM_TOL))
    y.copy_(torch.full_like(y, 7.0, dtype=torch.float32))
    assert bool((ybuf.float() == 7.0).all())


@pytest.mark.parametrize("cols", [1, 2, 7, 8, 31, 32, 64, 100, 255, 256, 264, 320, 1000, 1024, 1032, 2048, 2049, 4096,
                                  5119, 8192, 8200, 10000, 16384, 16392, 32760, 32767, 32768])
@pytest.mark.parametrize("rows", [1, 3, 300])
def test_norm_extents(cuda_torch, rows, cols):
    run_norm(cuda_torch, rows, cols, yt="e4m3", mode="row", seed=cols)
    run_norm(cuda_torch, rows, cols, yt="bf16", residual=False, keep_sum=False, seed=cols + 1)


@pytest.mark.parametrize("cols", [4097, 4104, 5120, 5121, 5128, 6143, 6144, 6145, 7000, 7168, 7169, 7176])
@pytest.mark.parametrize("rows", [2, 400])
def test_norm_teams_between_powers_of_two(cuda_torch, rows, cols):
    run_norm(cuda_torch, rows, cols, yt="e4m3", mode="row", seed=cols)


@pytest.mark.parametrize("xt,yt,rt", list(itertools.product(["f32", "f16", "bf16"], ["f32", "f16", "bf16", "e4m3"],
                                                        ["f32", "f16", "bf16"])))
def test_norm_types(cuda_torch, xt, yt, rt):
    wt = {"f32": "f16", "f16": "bf16", "bf16": "f32"}[xt]
    for cols in (328, 333, 2048):
        for mode in ("row", "tensor") if yt == "e4m3" else (None,):
            run_norm(cuda_torch, 37, cols, xt, yt, rt, wt, mode, seed=cols)


@pytest.mark.parametrize("residual,keep_sum,weight", list(itertools.product([False, True], repeat=3)))
def test_norm_optional_operands(cuda_torch, residual, keep_sum, weight):
    for cols in (96, 4096, 4097):
        run_norm(cuda_torch, 5, cols, "f16", "f32", "f32", "f32", None, residual, keep_sum, weight)


@pytest.mark.parametrize("offset", [0, 1, 3, 8])
@pytest.mark.parametrize("strides", [(0, 0, 0, 0), (528, 520, 544, 536), (521, 0, 0, 0), (0, 523, 0, 0), (0, 0, 525, 0),
                                     (0, 0, 0, 527)])
def test_norm_strides_and_offsets(cuda_torch, strides, offset):
    for yt, mode in (("e4m3", "row"), ("f16", None)):
        run_norm(cuda_torch, 9, 512, "bf16", yt, "f32", mode=mode, strides=strides, offset=offset)


def test_norm_rows_past_32_bits(cuda_torch):
    torch = cuda_torch
    rows, cols, stride = 1100, 256, 1 << 22  # 4.6 G elements from the first row to the last
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    run_norm(torch, rows, cols, strides=(stride, 0, stride, 0), keep_sum=True)
    torch.cuda.empty_cache()
    run_norm(torch, rows, cols, residual=False, keep_sum=False, yt="e4m3", mode="row", strides=(0, 0, 0, stride))
    torch.cuda.empty_cache()


def test_norm_many_rows(cuda_torch):
    run_norm(cuda_torch, 70001, 48, yt="e4m3", mode="row")
    run_norm(cuda_torch, 200001, 8, "f16", "f16", "f16")


def test_norm_in_place(cuda_torch):
    torch = cuda_torch
    for cols in (40, 77, 4096, 20000):
        x = torch.randn(11, cols, device="cuda").bfloat16()
        r = torch.randn(11, cols, device="cuda").bfloat16()
        h, v = norm_want(torch, x, r, None, 1e-6)
        # the sum in place of the residual, the result in place of x
        x1, r1 = x.clone(), r.clone()
        fx.rms_norm_dev(ptr(x1), ptr(x1), 11, cols, residual_ptr=ptr(r1), sum_ptr=ptr(r1), stream=stream(torch))
        check_close(torch, x1, v, HALF["bf16"] + NORM_TOL, 0)
        check_close(torch, r1, h, HALF["bf16"] + 2 * U, TINY["bf16"])
        # the sum in place of x
        x2, y2 = x.clone(), torch.empty_like(x)
        fx.rms_norm_dev(ptr(x2), ptr(y2), 11, cols, residual_ptr=ptr(r), sum_ptr=ptr(x2), stream=stream(torch))
        assert torch.equal(x2, r1) and torch.equal(y2, x1)


@pytest.mark.parametrize("cols", [64, 100, 3000, 9000])
def test_norm_extreme_rows(cuda_torch, cols):
    torch = cuda_torch
    inf, nan = float("inf"), float("nan")
    x = torch.randn(10, cols, device="cuda")
    x[1] = 0.0
    x[2, 5] = inf
    x[3, 6] = nan
    x[4] *= 1e-22   # squares below f32's range: eps alone is left
    x[5] *= 1e25    # squares past f32's range
    x[6] = 3.0e38
    x[7, cols - 1] = -inf
    for yt, mode in (("f32", None), ("bf16", None), ("e4m3", "row"), ("e4m3", "tensor")):
        y = torch.empty(10, cols, dtype=tt(torch, yt), device="cuda")
        scale = torch.full((10,), 0.02, device="cuda") if mode else None
        fx.rms_norm_dev(ptr(x), ptr(y), 10, cols, "f32", yt, scale_ptr=ptr(scale), scale_mode=mode, eps=1e-6,
                        stream=stream(torch))
        torch.cuda.synchronize()
        _, v = norm_want(torch, x, None, None, 1e-6)
        got, fine = y.float(), [0, 1, 4, 5, 6, 8, 9]
        assert bool(got[fine].isfinite().all())
        assert bool(got[3].isnan().all())
        if mode == "row":
            assert bool(got[2].isnan().all()) and bool(got[7].isnan().all())
            assert bool(scale[[2, 3, 7]].isnan().all())
            sc = scale[fine].double()[:, None]
            check_close(torch, scale[fine], v[fine].abs().amax(1).clamp(min=1e-30) / 448, NORM_TOL, 0)
            check_close(torch, got[fine], v[fine] / sc, HALF["e4m3"] + NORM_TOL, TINY["e4m3"])
        else:
            for r, c in ((2, 5), (7, cols - 1)):
                assert bool(got[r, c].isnan()) and int(got[r].isnan().sum()) == 1 and got[r].nansum().item() == 0.0
            if mode is None:
                check_close(torch, got[fine], v[fine], HALF[yt] + NORM_TOL, TINY[yt])
            else:
                check_close(torch, got[fine], (v[fine] / 0.02).clamp(-448, 448), HALF["e4m3"] + NORM_TOL + U, TINY["e4m3"])


@pytest.mark.parametrize("xt", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(4, 100), (4, 4096), (300, 64), (300, 1024), (300, 8192)])
def test_norm_rows_near_zero(cuda_torch, rows, cols, xt):
    """1 / sqrt(eps) times the least row scale's reciprocal is past f32's range."""
    torch, eps = cuda_torch, 1e-12
    x = torch.zeros(rows, cols, dtype=tt(torch, xt), device="cuda")
    x[1::3] = (torch.arange(cols, device="cuda") % 15 - 7) * 2.0 ** -125  # v of some 1e-31, below the least maximum
    x[2::3] = torch.randn(cols, device="cuda").to(x.dtype)
    y = torch.empty(rows, cols, dtype=tt(torch, "e4m3"), device="cuda")
    scale = torch.zeros(rows, device="cuda")
    fx.rms_norm_dev(ptr(x), ptr(y), rows, cols, xt, "e4m3", scale_ptr=ptr(scale), scale_mode="row", eps=eps, stream=stream(torch))
    _, v = norm_want(torch, x, None, None, eps)
    check_close(torch, scale, v.abs().amax(1).clamp(min=1e-30) / 448, NORM_TOL, 0)
    assert bool((y[0::3].float() == 0).all())
    check_close(torch, y.float(), v / scale.double()[:, None], HALF["e4m3"] + NORM_TOL, TINY["e4m3"])


# ---- 4-bit weights ----------------------------------------------------------------------------------------------


def unpack(torch, codes, scales, zeros, group):
    n, k = codes.shape[0], codes.shape[1] * 2
    c = torch.stack((codes & 15, codes >> 4), 2).view(n, k // group, group).double()
    z = zeros.double()[..., None] if zeros is not None else 8.0
    return ((c - z) * scales.double()[..., None]).view(n, k)


def quantize_want(torch, w, group, st, zeros):
    """The definition, in f64 where f32's correctly rounded quotients cannot differ from it in what is rounded next."""
    n, k = w.shape
    v = w.float().view(n, k // group, group)
    if zeros:
        lo, hi = v.amin(2).clamp(max=0), v.amax(2).clamp(min=0)
        s = (hi - lo) / torch.full_like(hi, 15.0)
    else:
        s = v.abs().amax(2) / torch.full_like(v[..., 0], 7.0)
    s = s.to(tt(torch, st)).float()
    z = torch.full_like(s, 8.0)
    if zeros:
        z = torch.where(s > 0, torch.round(-lo / s), torch.zeros_like(s)).clamp(0, 15)
    q = torch.where(s[..., None] > 0, torch.round(v / s[..., None]), torch.zeros_like(v)) + z[..., None]
    q = q.clamp(0, 15).to(torch.uint8).view(n, k)
    return q[:, 0::2] | (q[:, 1::2] << 4), s, z.to(torch.uint8)


def quantize(torch, w, wt, group, st, zeros, w_stride=0):
    n, k = w.shape
    codes = torch.full((n + 1, k // 2), 0x5a, dtype=torch.uint8, device="cuda")
    scales = torch.full((n + 1, k // group), 3.0, dtype=tt(torch, st), device="cuda")
    zp = torch.full((n + 1, k // group), 99, dtype=torch.uint8, device="cuda") if zeros else None
    fx.w4_quantize_dev(ptr(w), n, k, group, ptr(codes), ptr(scales), ptr(zp), wt, st, w_stride, stream(torch))
    torch.cuda.synchronize()
    # the row behind the last is as it was
    assert bool((codes[n] == 0x5a).all()) and bool((scales[n] == 3.0).all()) and (zp is None or bool((zp[n] == 99).all()))
    return codes[:n], scales[:n], zp[:n] if zeros else None


@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (3, 64, 64), (5, 96, 32), (7, 160, 160), (33, 1088, 32), (64, 4096, 128),
                                       (17, 1344, 448), (2, 8192, 8192), (129, 768, 256), (1000, 192, 64)])
@pytest.mark.parametrize("wt,st,zeros", [("f32", "f16", False), ("bf16", "bf16", True), ("f16", "f32", True),
                                         ("f32", "f32", False), ("bf16", "f16", True)])
def test_quantize_and_back(cuda_torch, n, k, group, wt, st, zeros):
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(n + k)
    for stride, offset in ((0, 0), (k + 8, 8), (k + 3, 1)):
        _, w = rows_of(torch, n, k, tt(torch, wt), stride, offset)
        w.copy_(torch.randn(n, k, generator=g, device="cuda") * 0.05)
        w[0, :32] = 0.0  # a group of zeros where groups are 32 long
        codes, scales, zp = quantize(torch, w, wt, group, st, zeros, stride)
        want = quantize_want(torch, w, group, st, zeros)
        assert torch.equal(scales.float(), want[1])
        assert torch.equal(codes, want[0])
        assert zp is None or torch.equal(zp, want[2])
        for ot in ("f32", "f16", "bf16"):
            obuf, out = rows_of(torch, n, k, tt(torch, ot), stride, offset, 7.0)
            fx.w4_dequantize_dev(ptr(codes), ptr(scales), n, k, group, ptr(out), ptr(zp), ot, st, stride, stream(torch))
            torch.cuda.synchronize()
            # scale * (code - zero) has at most 24 + 5 bits: f32 rounds once more before the 16-bit types
            check_close(torch, out, unpack(torch, codes, scales, zp, group), HALF[ot] + U, TINY[ot])
            out.fill_(7.0)
            assert bool((obuf == 7.0).all())


@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_extreme_groups(cuda_torch, zeros):
    torch = cuda_torch
    w = torch.randn(9, 64, device="cuda")
    w[0] = 0.0
    w[1, 3] = float("nan")
    w[2] = float("nan")
    w[3] *= 1e-12   # the f16 scale rounds to zero
    w[4] *= 1e9     # the f16 scale saturates
    w[5, 9] = float("inf")
    w[6, 9] = float("-inf")
    w[7] = 0.5      # all of one sign
    w[8] = -0.5
    codes, scales, zp = quantize(torch, w, "f32", 32, "f16", zeros)
    got = unpack(torch, codes, scales, zp, 32)
    assert bool(scales.isfinite().all()) and bool(got.isfinite().all())
    assert bool((got[[0, 2, 3]] == 0).all()) and got[1, 3].item() == 0.0
    assert bool((scales[4] == 65504).all()) and got[5, 9].item() > 4e5 and got[6, 9].item() < -4e5
    plain = w.clone()
    plain[1, 3] = 0.0
    half = scales.double().repeat_interleave(32, 1) * 0.5
    for r in (1, 7, 8):
        # the end points of a range move with the rounded zero point: by half a step at most, on top of half a step
        assert bool(((got[r] - plain[r].double()).abs() <= half[r] * (2.0 if zeros else 1.0) * (1 + 2.0 ** -8)).all())
    out = torch.empty(9, 64, device="cuda")
    fx.w4_dequantize_dev(ptr(codes), ptr(scales), 9, 64, 32, ptr(out), ptr(zp), "f32", "f16", stream=stream(torch))
    assert torch.equal(out.double(), got)


def test_quantize_past_32_bits(cuda_torch):
    torch = cuda_torch
    n, k, stride = 1100, 64, 1 << 22
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB of free device memory")
    _, w = rows_of(torch, n, k, torch.bfloat16, stride)
    w.copy_(torch.randn(n, k, device="cuda"))
    codes, scales, _ = quantize(torch, w, "bf16", 32, "f16", False, stride)
    assert torch.equal(codes, quantize_want(torch, w, 32, "f16", False)[0])
    fx.w4_dequantize_dev(ptr(codes), ptr(scales), n, k, 32, ptr(w), w_type="bf16", w_stride=stride, stream=stream(torch))
    check_close(torch, w, unpack(torch, codes, scales, None, 32), HALF["bf16"] + U, TINY["bf16"])
    del w
    torch.cuda.empty_cache()


# ---- the linear layer -------------------------------------------------------------------------------------------


def make_layer(torch, n, k, group, st, zeros, g, exact):
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    if exact:
        scales = 2.0 ** torch.randint(-9, -5, (n, k // group), generator=g, device="cuda").float()
    else:
        scales = (torch.rand(n, k // group, generator=g, device="cuda") + 0.25) * 0.02
    zp = torch.randint(0, 16, (n, k // group), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return codes, scales.to(tt(torch, st)), zp


def run_linear(torch, rows, n, k, group, xt="bf16", yt="bf16", st="f16", zeros=False, bias=False, mode=None, exact=True,
               xs=0, ys=0, offset=0, seed=0, given=None):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * rows + n)
    codes, scales, zp = make_layer(torch, n, k, group, st, zeros, g, exact)
    mode = mode or ("row" if xt == "e4m3" else None)
    if exact:
        x0 = torch.randint(-4, 5, (rows, k), generator=g, device="cuda").float()
    else:
        x0 = torch.randn(rows, k, generator=g, device="cuda")
    xbuf, x = rows_of(torch, rows, k, tt(torch, xt), xs, offset)
    x.copy_(x0)
    b = sc = None
    if bias:
        b = torch.randint(-8, 9, (n,), generator=g, device="cuda").float() / 8
    if mode:
        sc = 2.0 ** torch.randint(-2, 3, (rows if mode == "row" else 1,), generator=g, device="cuda").float()
        if not exact:
            sc = sc * 0.77
    ybuf, y = rows_of(torch, rows, n, tt(torch, yt), ys, offset, 7.0)
    fx.w4_linear_dev(ptr(x), ptr(y), rows, n, k, group, ptr(codes), ptr(scales), ptr(zp), xt, yt, st, xs, ys, ptr(sc),
                     mode, ptr(b), stream(torch))
    torch.cuda.synchronize()
    xv = x.float().double()
    if sc is not None:
        xv = xv * sc.double()[:, None]
    w = unpack(torch, codes, scales, zp, group)
    want = xv @ w.t()
    if b is not None:
        want = want + b.double()
    if exact:
        assert torch.equal(y, want.float().to(y.dtype))
    else:
        half_w = HALF["bf16" if xt == "bf16" else "f16"]
        tol = 4 * half_w * (xv.square() @ w.square().t()).sqrt() + k / 16 * 2.0 ** -22 * (xv.abs() @ w.abs().t())
        err = (y.double() - want).abs()
        lim = tol * (1 + HALF[yt]) + (HALF[yt] + 4 * U) * want.abs() + TINY[yt]
        assert bool((err <= lim).all()), ((err - lim).max().item(), err.max().item())
    y.fill_(7.0)
    assert bool((ybuf == 7.0).all())  # nothing outside the rows was written


ROWS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 48, 64, 65, 96, 127, 128, 129, 192, 255, 256, 257, 300, 513]


@pytest.mark.parametrize("rows", ROWS)
def test_linear_rows(cuda_torch, rows):
    for n, k, group in ((200, 512, 128), (65, 1120, 32), (384, 256, 64)):
        run_linear(cuda_torch, rows, n, k, group, zeros=rows % 2 == 0, bias=rows % 3 == 0)
        run_linear(cuda_torch, rows, n, k, group, "f16", "f16", zeros=rows % 2 == 1, exact=False)


@pytest.mark.parametrize("n", [1, 2, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000])
def test_linear_outputs(cuda_torch, n):
    for rows in (1, 6, 13, 40, 150):
        run_linear(cuda_torch, rows, n, 384, 128, zeros=n % 2 == 0, bias=True)
        run_linear(cuda_torch, rows, n, 384, 32, "e4m3", "f16", zeros=n % 2 == 1)


@pytest.mark.parametrize("k,group", [(32, 32), (64, 32), (64, 64), (96, 32), (96, 96), (128, 128), (160, 32), (192, 64),
                                     (224, 224), (288, 96), (352, 32), (480, 160), (1024, 1024), (1120, 224), (2080, 32),
                                     (4096, 4096), (4704, 32), (5120, 256), (8192, 64), (16384, 128), (28672, 128)])
def test_linear_inner(cuda_torch, k, group):
    for rows in (1, 5, 12, 35, 140):
        run_linear(cuda_torch, rows, 144, k, group, zeros=rows % 2 == 0)
        run_linear(cuda_torch, rows, 50, k, group, "e4m3", "bf16", zeros=rows % 2 == 1, exact=False)


@pytest.mark.parametrize("xt,yt,st,zeros,mode", [
    (xt, yt, st, z, m) for xt in ("f16", "bf16", "e4m3") for yt in ("f16", "bf16") for st in ("f32", "f16", "bf16")
    for z in (False, True) for m in (("row", "tensor") if xt == "e4m3" else (None,))])
def test_linear_types(cuda_torch, xt, yt, st, zeros, mode):
    for rows in (1, 8, 20, 130):
        run_linear(cuda_torch, rows, 136, 640, 64, xt, yt, st, zeros, True, mode, exact=False)
        run_linear(cuda_torch, rows, 136, 640, 32, xt, yt, st, zeros, True, mode)


@pytest.mark.parametrize("xs,ys,offset", [(0, 0, 1), (520, 0, 0), (520, 264, 8), (513, 0, 0), (0, 251, 0), (515, 253, 3),
                                          (0, 250, 2), (514, 256, 4)])
def test_linear_strides_and_offsets(cuda_torch, xs, ys, offset):
    for rows, xt in itertools.product((1, 6, 20, 70, 200), ("bf16", "e4m3")):
        run_linear(cuda_torch, rows, 250, 512, 64, xt, "bf16", xs=xs, ys=ys, offset=offset)


def test_linear_large(cuda_torch):
    run_linear(cuda_torch, 1, 28672, 8192, 128, "f16", "f16", exact=False)
    run_linear(cuda_torch, 2000, 1500, 4096, 128, exact=False)
    run_linear(cuda_torch, 1500, 3000, 2048, 64, "e4m3", "f16", zeros=True, bias=True)


@pytest.mark.parametrize("xt,zeros,group,offset", [("bf16", False, 128, 0), ("f16", True, 64, 0), ("e4m3", False, 128, 0),
                                                   ("e4m3", True, 32, 0), ("e4m3", False, 64, 1), ("bf16", True, 32, 1)])
def test_linear_tiles_that_fill_the_gpu(cuda_torch, xt, zeros, group, offset):
    """Tiles of 256 outputs: more of them than SMs, ragged at both edges, rows by TMA, widened, and value by value."""
    run_linear(cuda_torch, 2005, 5003, 1120 if group == 32 else 1152, group, xt, "f16" if xt == "f16" else "bf16", zeros=zeros,
               bias=True, offset=offset)


@pytest.mark.parametrize("xt,offset", [("bf16", 0), ("f16", 1), ("e4m3", 0), ("e4m3", 1)])
def test_linear_inputs_over_a_cluster(cuda_torch, xt, offset):
    """One tile of outputs and many inputs: a cluster shares it, some of its blocks without inputs of their own."""
    for rows, k in ((9, 28672), (70, 8192 + 256), (250, 9 * 1024), (16, 4 * 1024 + 32 * 8)):
        run_linear(cuda_torch, rows, 100, k, 32, xt, "bf16", zeros=True, bias=True, offset=offset)


@pytest.mark.parametrize("tiles", [9, 15, 16, 22, 23, 26, 27, 33, 34, 45, 46, 74, 75])
def test_linear_clusters_of_every_size(cuda_torch, tiles):
    """Tiles of 128 outputs, shared by clusters of as many blocks as the GPU runs at once; the last tile is a part."""
    run_linear(cuda_torch, 20, tiles * 128 - 5, 3584, 128, "bf16", "bf16", zeros=True, bias=True)
    run_linear(cuda_torch, 130, tiles * 128 - 64, 2176, 64, "e4m3", "f16", mode="row")


def test_linear_rows_past_32_bits(cuda_torch):
    torch = cuda_torch
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    for rows, n in ((1100, 128),):
        run_linear(torch, rows, n, 128, 32, xs=1 << 22)
        torch.cuda.empty_cache()
        run_linear(torch, rows, n, 128, 32, "f16", ys=1 << 22)
        torch.cuda.empty_cache()


@pytest.mark.parametrize("xt", ["f16", "bf16", "e4m3"])
def test_linear_wide_range_of_scales(cuda_torch, xt):
    """Scales far from one and unequal by powers of two within a row: f32 scales up to 2^60 and down to 2^-60."""
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(5)
    n, k, group = 96, 512, 64
    codes, _, zp = make_layer(torch, n, k, group, "f32", True, g, True)
    row = torch.randint(-55, 56, (n, 1), generator=g, device="cuda").float()
    scales = 2.0 ** (row + torch.randint(-5, 6, (n, k // group), generator=g, device="cuda").float())
    for rows in (1, 8, 16, 30, 129):
        x = torch.randint(-4, 5, (rows, k), generator=g, device="cuda").float().to(tt(torch, xt))
        sc = torch.ones(rows, device="cuda") if xt == "e4m3" else None
        y = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
        fx.w4_linear_dev(ptr(x), ptr(y), rows, n, k, group, ptr(codes), ptr(scales), ptr(zp), xt, "bf16", "f32",
                         x_scale_ptr=ptr(sc), x_scale_mode="row" if xt == "e4m3" else None, stream=stream(torch))
        torch.cuda.synchronize()
        want = x.double() @ unpack(torch, codes, scales, zp, group).t()
        assert torch.equal(y, want.float().bfloat16())


@pytest.mark.parametrize("rows", [1, 8, 12, 20, 130])
def test_linear_nonfinite_rows_stay_apart(cuda_torch, rows):
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(6)
    n, k, group = 200, 256, 32
    codes, scales, zp = make_layer(torch, n, k, group, "f16", False, g, True)
    x = torch.randint(-4, 5, (rows + 2, k), generator=g, device="cuda").bfloat16()
    clean = x.clone()
    x[0, 5] = float("nan")
    x[rows] = float("nan")  # behind the last row
    y = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    fx.w4_linear_dev(ptr(x), ptr(y), rows, n, k, group, ptr(codes), ptr(scales), stream=stream(torch))
    torch.cuda.synchronize()
    assert bool(y[0].isnan().all())
    want = clean[:rows].double() @ unpack(torch, codes, scales, zp, group).t()
    assert torch.equal(y[1:], want[1:].float().bfloat16())
    # a scale of infinity or NaN reaches its own output only
    scales[3, 1] = float("inf")
    scales[4, 0] = float("nan")
    fx.w4_linear_dev(ptr(clean), ptr(y), rows, n, k, group, ptr(codes), ptr(scales), stream=stream(torch))
    torch.cuda.synchronize()
    others = [i for i in range(n) if i not in (3, 4)]
    assert torch.equal(y[:, others], want.float().bfloat16()[:, others])
    assert not bool(y[:, 3].isfinite().any()) and bool(y[:, 4].isnan().all())


# ---- used together ----------------------------------------------------------------------------------------------


class Block:
    """norm -> 8-bit linear, its weights quantised on the device from f32."""

    def __init__(self, torch, rows, k, n, group, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.torch, self.rows, self.k, self.n, self.group = torch, rows, k, n, group
        self.w = torch.randn(n, k, generator=g, device="cuda") / k ** 0.5
        self.x = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
        self.r = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
        self.gain = (torch.rand(k, generator=g, device="cuda") + 0.5).bfloat16()
        self.codes = torch.empty(n, k // 2, dtype=torch.uint8, device="cuda")
        self.scales = torch.empty(n, k // group, dtype=torch.float16, device="cuda")
        self.zeros = torch.empty(n, k // group, dtype=torch.uint8, device="cuda")
        self.sum = torch.empty_like(self.x)
        self.q = torch.empty(rows, k, dtype=torch.float8_e4m3fn, device="cuda")
        self.qs = torch.empty(rows, device="cuda")
        self.y = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")

    def quantize(self):
        fx.w4_quantize_dev(ptr(self.w), self.n, self.k, self.group, ptr(self.codes), ptr(self.scales), ptr(self.zeros),
                           stream=stream(self.torch))

    def step(self):
        fx.rms_norm_dev(ptr(self.x), ptr(self.q), self.rows, self.k, "bf16", "e4m3", ptr(self.gain), residual_ptr=ptr(self.r),
                        sum_ptr=ptr(self.sum), scale_ptr=ptr(self.qs), scale_mode="row", stream=stream(self.torch))
        fx.w4_linear_dev(ptr(self.q), ptr(self.y), self.rows, self.n, self.k, self.group, ptr(self.codes), ptr(self.scales),
                         ptr(self.zeros), "e4m3", "bf16", x_scale_ptr=ptr(self.qs), x_scale_mode="row",
                         stream=stream(self.torch))

    def check(self):
        torch = self.torch
        want_codes, want_scales, want_zeros = quantize_want(torch, self.w, self.group, "f16", True)
        assert torch.equal(self.codes, want_codes) and torch.equal(self.zeros, want_zeros)
        _, v = norm_want(torch, self.x, self.r, self.gain, 1e-6)
        q = self.q.float().double() * self.qs.double()[:, None]
        # half a step relative, or half the smallest step where the value is subnormal
        assert bool(((q - v).abs() <= (HALF["e4m3"] + NORM_TOL) * v.abs() + 2.0 ** -10 * 1.01 * self.qs.double()[:, None]).all())
        w = unpack(torch, self.codes, self.scales, self.zeros, self.group)
        want = q @ w.t()
        tol = 4 * HALF["f16"] * (q.square() @ w.square().t()).sqrt() + self.k / 16 * 2.0 ** -22 * (q.abs() @ w.abs().t())
        assert bool(((self.y.double() - want).abs() <= tol * 1.01 + (HALF["bf16"] + 4 * U) * want.abs()).all())


@pytest.mark.parametrize("rows,k,n,group", [(1, 1024, 512, 128), (4, 2048, 1000, 64), (20, 512, 264, 32), (200, 768, 384, 256)])
def test_block_of_calls(cuda_torch, rows, k, n, group):
    b = Block(cuda_torch, rows, k, n, group)
    b.quantize()
    b.step()
    cuda_torch.cuda.synchronize()
    b.check()


@pytest.mark.parametrize("rows", [1, 6, 40, 200])
def test_captured_replayed_and_side_by_side(cuda_torch, rows):
    """Two graphs of the same calls on two streams at once, replayed on new inputs, with eager calls between."""
    torch = cuda_torch
    blocks = [Block(torch, rows, 1024, 640, 64, seed=s) for s in range(3)]
    streams = [torch.cuda.Stream() for _ in blocks]
    graphs = []
    torch.cuda.synchronize()
    for b, st in zip(blocks[:2], streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            b.quantize()
            b.step()
        graphs.append(g)
    for turn in range(3):
        for i, b in enumerate(blocks):
            b.x.copy_(torch.randn_like(b.x.float()) * (turn + 1))
            b.w.copy_(torch.randn_like(b.w) * 0.1)
        torch.cuda.synchronize()
        for _ in range(4):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
            with torch.cuda.stream(streams[2]):
                blocks[2].quantize()
                blocks[2].step()
        torch.cuda.synchronize()
        for b in blocks:
            b.check()


def test_repeatable(cuda_torch):
    """The same call gives the same bits: no sum's order changes from run to run."""
    torch = cuda_torch
    for rows in (1, 8, 20, 100, 300):
        b = Block(torch, rows, 4096, 700, 128)
        b.quantize()
        b.step()
        first = [t.clone() for t in (b.sum, b.q.view(torch.uint8), b.qs, b.y)]
        for _ in range(5):
            b.step()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(first, (b.sum, b.q.view(torch.uint8), b.qs, b.y)))


def test_no_wait_gave_up(cuda_torch):
    run_linear(cuda_torch, 3, 64, 256, 64)
    run_linear(cuda_torch, 30, 64, 256, 64)
    fx.w4_device_status(0)
    with pytest.raises(fx.FxError):
        fx.w4_device_status(-1)


def test_host_pointers_are_refused(cuda_torch):
    torch = cuda_torch
    d = torch.zeros(64, 64, device="cuda", dtype=torch.bfloat16)
    h = torch.zeros(64, 64, dtype=torch.bfloat16)
    with pytest.raises(fx.FxError) as e:
        fx.rms_norm_dev(ptr(h), ptr(d), 4, 64)
    assert e.value.code == fx.FX_INVALID_ARGUMENT and "device memory" in str(e.value)
    with pytest.raises(fx.FxError) as e:
        fx.w4_linear_dev(ptr(d), ptr(d[8:]), 4, 8, 64, 32, ptr(h), ptr(d))
    assert e.value.code == fx.FX_INVALID_ARGUMENT
    run_norm(torch, 3, 64)  # and the next call is served


def test_other_device(cuda_torch):
    torch = cuda_torch
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    x = torch.randn(5, 256, device="cuda:1").bfloat16()
    y = torch.empty_like(x)
    with torch.cuda.device(0):
        fx.rms_norm_dev(ptr(x), ptr(y), 5, 256)
        assert torch.cuda.current_device() == 0
    torch.cuda.synchronize(1)
    _, v = norm_want(torch, x, None, None, 1e-6)
    check_close(torch, y, v, HALF["bf16"] + NORM_TOL, TINY["bf16"])
    z = torch.empty(5, 256, device="cuda:0", dtype=torch.bfloat16)
    with pytest.raises(fx.FxError):
        fx.rms_norm_dev(ptr(x), ptr(z), 5, 256)
