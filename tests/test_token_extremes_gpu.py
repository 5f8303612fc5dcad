"""The token-row calls at the ends of f32's range, where a sum, a difference or a reciprocal of the formulas' leaves it
although the result does not."""
import pytest
import test_token_gpu as base
from test_token_gpu import HALF, NORM_TOL, TINY, ptr, stream, tt

import fenix_b200 as fx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wt", ["f32", "bf16"])
@pytest.mark.parametrize("st", ["f32", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128, 512])
def test_quantize_ranges_past_f32(cuda_torch, wt, st, group):
    """hi - lo is past f32's largest value, (hi - lo) / 15 is not."""
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(group)
    n, k = 7, 512
    w = ((2 * torch.rand(n, k, generator=g, device="cuda") - 0.94) * 3.1e38).to(tt(torch, wt))
    assert bool(w.isfinite().all())
    w.view(n, k // group, group)[:, :, 3] = -2.9e38
    w.view(n, k // group, group)[:, :, 7] = 3.2e38
    w[1] *= 0.01  # and an ordinary row between
    codes, scales, zp = base.quantize(torch, w, wt, group, st, True)
    v = w.double().view(n, k // group, group)
    lo, hi = v.amin(2).clamp(max=0), v.amax(2).clamp(min=0)
    want = ((hi / 2).float() - (lo / 2).float()) / torch.full_like(scales, 7.5, dtype=torch.float32)  # f32's quotient
    want = want.to(tt(torch, st))
    assert torch.equal(scales, want)
    s = scales.double()
    z = torch.round(-lo / s).clamp(0, 15)
    assert torch.equal(zp.double(), z)
    q = torch.round(v / s[..., None])
    near = ((v / s[..., None]).frac().abs() - 0.5).abs() < 2.0 ** -20  # quotients that f32 may round either way
    got = torch.stack((codes & 15, codes >> 4), 2).view(n, k // group, group).double()
    assert bool(((got - (q + z[..., None]).clamp(0, 15)).abs() <= near).all())  # by one there, by none elsewhere


@pytest.mark.parametrize("rows", [1, 5, 1000])
@pytest.mark.parametrize("yt", ["f32", "bf16"])
def test_norm_eps_and_squares_past_f32_together(cuda_torch, rows, yt):
    torch = cuda_torch
    eps = 2.9e38
    for cols in (1, 2, 64):
        x = torch.full((rows, cols), 1.6e19 / cols ** 0.5, device="cuda")
        x[::2] *= -0.9
        y = torch.empty(rows, cols, dtype=tt(torch, yt), device="cuda")
        fx.rms_norm_dev(ptr(x), ptr(y), rows, cols, "f32", yt, eps=eps, stream=stream(torch))
        torch.cuda.synchronize()
        eps32 = float(torch.tensor(eps, dtype=torch.float32))
        _, v = base.norm_want(torch, x, None, None, eps32)
        base.check_close(torch, y, v, HALF[yt] + NORM_TOL, TINY[yt])


@pytest.mark.parametrize("rows,cols", [(3, 100), (2, 4096), (600, 64), (900, 2048)])
@pytest.mark.parametrize("scale", [2.0 ** -128, 2.0 ** -149, 2.0 ** -127 * 1.5])
def test_norm_tensor_scales_whose_reciprocal_is_past_f32(cuda_torch, rows, cols, scale):
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(rows, cols, generator=g, device="cuda").bfloat16()
    x[:, ::5] = 0.0
    w = torch.full((cols,), 2.0 ** -125, device="cuda")
    w[:cols // 2] = 2.0
    sc = torch.tensor([scale], device="cuda", dtype=torch.float64).float()
    y = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device="cuda")
    fx.rms_norm_dev(ptr(x), ptr(y), rows, cols, "bf16", "e4m3", ptr(w), "f32", 1e-5, scale_ptr=ptr(sc), scale_mode="tensor",
                    stream=stream(torch))
    torch.cuda.synchronize()
    _, v = base.norm_want(torch, x, None, w, float(torch.tensor(1e-5, dtype=torch.float32)))
    # v itself comes close to f32's smallest normal value: half a subnormal step of it, over the scale, is added
    want = (v / sc.double()).clamp(-448, 448)
    base.check_close(torch, y.float(), want, HALF["e4m3"] + NORM_TOL, TINY["e4m3"] + 2.0 ** -150 / scale * (1 + HALF["e4m3"]))
