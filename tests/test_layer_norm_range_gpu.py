"""The layer norm at the ends of f32's range."""
import pytest

import fenix_b200 as fx
from test_layer_norm_gpu import TOP, check_norm, dtype, norm_want, within
from test_token_gpu import HALF, U, ptr, stream, tt

pytestmark = pytest.mark.gpu

FORMS = [("f32", None), ("bf16", None), ("e4m3", "row"), ("e4m3", "tensor"), ("i8", "row"), ("i8", "tensor")]


def run(torch, x, xt, yt, mode, bias):
    rows, cols = x.shape
    y = torch.empty(rows, cols, dtype=dtype(torch, yt), device="cuda")
    scale = torch.full((rows if mode == "row" else 1,), 0.02, device="cuda") if mode else None
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    fx.layer_norm_dev(ptr(x), ptr(y), rows, cols, xt, yt, None, ptr(bias), "f32", 1e-6, mean_ptr=ptr(mean), rstd_ptr=ptr(rstd),
                      scale_ptr=ptr(scale), scale_mode=mode, stream=stream(torch))
    torch.cuda.synchronize()
    return y, scale, mean, rstd


@pytest.mark.parametrize("xt,rows,cols", [("f32", 4, 3), ("f32", 4, 64), ("f32", 4, 300), ("f32", 4, 1000), ("f32", 700, 333),
                                          ("bf16", 5, 64), ("bf16", 5, 77), ("bf16", 3000, 64), ("bf16", 9000, 200)])
def test_differences_past_the_range(cuda_torch, xt, rows, cols):
    """A sum inside f32's range and a difference from the mean past it: such a row is NaN throughout, and no other."""
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(rows, cols, generator=g, device="cuda")
    top = torch.finfo(tt(torch, xt)).max
    bad = [1, rows - 1]
    for i, sign in zip(bad, (1, -1)):
        x[i] = 0.0
        x[i, 0], x[i, 1], x[i, 2] = sign * top, -sign * top, -sign * 2.9e38
    x = x.to(tt(torch, xt))
    assert bool(((x[bad].float() - (x[bad].double().sum(1, keepdim=True) / cols).float()).isinf()).any(1).all())
    bias = torch.full((cols,), 0.5, device="cuda")
    others = [i for i in range(rows) if i not in bad]
    for yt, mode in FORMS:
        y, scale, mean, rstd = run(torch, x, xt, yt, mode, bias)
        assert bool(rstd[bad].isnan().all()) and not bool(mean[bad].isfinite().any())
        assert bool((y[bad] == 0).all() if yt == "i8" else y[bad].float().isnan().all())
        assert mode != "row" or (bool(scale[bad].isnan().all()) and bool(scale[others].isfinite().all()))
        assert bool(y[others].float().isfinite().all()) and bool(rstd[others].isfinite().all())


ALIKE = [(3, 7), (3, 100), (3, 333), (3, 1000), (3, 4097), (3, 12345), (3, 30001), (9000, 96), (9000, 200), (9000, 328), (3000, 1000),
         (3000, 1536), (2600, 5000), (1500, 7000), (900, 12000)]


@pytest.mark.parametrize("xt", ["f32", "bf16"])
@pytest.mark.parametrize("v", [1.0, -1e6, 1e8, 1e10, -1e14, 1e20, 1e30, -3e38])
def test_rows_all_alike(cuda_torch, xt, v):
    """Values all alike are as far from their mean as it is off, c, whatever their size: the squares left about it are rounding, at most
    c^2 2^-17 (80 roundings), and c is brought down to where c^2 is within those and eps, so (2^-17 as often as need be) c r <= 1. Results are
    off by (1 + 2^-23) c - c and two roundings, 80 u c r at most in the sum's place: 100 u. rstd by 2^-18 and 8 u; 5 u |v| for the mean is
    a rounding for each time that it is made better, which is some 8 times at most: 10 u |v|."""
    torch = cuda_torch
    for rows, cols in ALIKE:
        x = torch.full((rows, cols), v, device="cuda").to(tt(torch, xt))
        bias = torch.full((cols,), 0.52, device="cuda")
        for yt, mode in FORMS:
            y, scale, mean, rstd = run(torch, x, xt, yt, mode, bias)
            if mode is None:
                within(y, bias.double(), torch.full_like(y, 100 * U + HALF[yt], dtype=torch.float64))
            else:
                assert bool((y.float() == (26.0 if mode == "tensor" else TOP[yt])).all())
            if mode == "row":
                within(scale, (bias[:1] / TOP[yt]).double(), torch.full_like(scale, 200 * U / TOP[yt], dtype=torch.float64))
            within(mean, x[:, 0].double(), 10 * U * x[:, 0].double().abs())
            within(rstd, torch.full_like(rstd, 1e3, dtype=torch.float64), torch.full_like(rstd, 1e3 * (2.0 ** -18 + 8 * U), dtype=torch.float64))


@pytest.mark.parametrize("v", [1e8, -1e14, 1e20, 2e38])
def test_rows_nearly_alike(cuda_torch, v):
    """f32 rows far from zero whose values differ in their last bits. t = h - mean is exact (neighbours), t - off is rounded once, and off^2 is no
    larger than the variance: it is off by 84 u, and as much by the cancellation, twice over (u of twice the variance and of off^2), its root by
    half: |z| 90 u. The mean's correction, 82 u of the mean magnitude of at most 2 standard deviations, and t's and off's roundings: 170 u."""
    torch = cuda_torch
    for rows, cols in ((3, 100), (3, 1000), (3, 4096), (3, 9001), (700, 1536)):
        g = torch.Generator(device="cuda").manual_seed(cols)
        x = torch.full((rows, cols), v, device="cuda")
        x = torch.where(torch.rand(rows, cols, generator=g, device="cuda") < 0.1, torch.nextafter(x, torch.zeros_like(x)), x)
        bias = torch.full((cols,), 0.5, device="cuda")
        var, m = torch.var_mean(x.double(), 1, correction=0, keepdim=True)
        z = (x.double() - m) / torch.sqrt(var + 1e-6)
        y, _, mean, rstd = run(torch, x, "f32", "f32", None, bias)
        within(y, z + 0.5, U * (200 + 110 * z.abs()))
        within(mean, m[:, 0], 10 * U * m[:, 0].abs())
        r = 1 / torch.sqrt(var[:, 0] + 1e-6)
        within(rstd, r, 110 * U * r + 2.0 ** -149)


@pytest.mark.parametrize("xt,rows,cols", [("f32", 5, 300), ("f32", 5, 4096), ("f32", 5, 4097), ("f32", 5, 20000), ("f32", 700, 1000),
                                          ("bf16", 5, 4096), ("bf16", 3000, 1024), ("bf16", 2600, 4096), ("bf16", 1300, 8192)])
def test_sums_past_the_range(cuda_torch, xt, rows, cols):
    """Rows of finite values whose sum is past f32's range: statistics and results of the definition, in the counts of the ordinary rows."""
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x[1] = 2.5e38 + 1e37 * torch.randn(cols, generator=g, device="cuda").clamp(-4, 4)
    x[2] = -1e38 * torch.rand(cols, generator=g, device="cuda") - 1e38
    x = x.to(tt(torch, xt))
    assert bool((x[1:3].double().sum(1).abs() > torch.finfo(torch.float32).max).all())
    bias = torch.full((cols,), 0.5, device="cuda")
    for yt, mode in FORMS:
        y, scale, mean, rstd = run(torch, x, xt, yt, mode, bias)
        check_norm(torch, x, None, None, bias, 1e-6, yt, y, scale, mode)
        _, m, r, _, _ = norm_want(torch, x, None, None, bias, 1e-6)
        top = x.double().abs().amax(1)
        within(mean, m, U * (3 * top + 84 / r))
        # an rstd below f32's normal numbers is rounded to a whole number of its smallest
        within(rstd, r, r * U * (50 * (1 + 80 * U * top * r) ** 2 + top * r) + 2.0 ** -149)
