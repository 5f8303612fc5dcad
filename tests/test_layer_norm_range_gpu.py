"""The layer norm at the ends of f32's range."""
import pytest

import fenix_b200 as fx
from test_layer_norm_gpu import dtype
from test_token_gpu import ptr, stream, tt

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
