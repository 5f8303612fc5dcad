"""The layer norm's 8-bit rows are those of its f32 rows: scale and codes of the definition's correctly rounded f32 quotients, bit
for bit what fx_i8_quantize makes of the f32 result."""
import itertools

import pytest

import fenix_b200 as fx
from test_layer_norm_gpu import TOP, dtype
from test_token_gpu import ptr, rows_of, stream, tt

pytestmark = pytest.mark.gpu


def scale_of(torch, v, yt):
    """Row scales as a tensor's quotient: torch multiplies by the reciprocal of a Python number."""
    return v.abs().amax(1, keepdim=True).clamp(min=1e-30) / torch.full((1,), TOP[yt], device="cuda")


def eighths(torch, v, scale, yt):
    q = v / scale
    return torch.round(q).clamp(-127, 127).to(torch.int8) if yt == "i8" else q.clamp(-448, 448).to(tt(torch, yt))


def both_ways(torch, rows, cols, xt, yt, mode, residual=True, weight=None, bias=None, offset=0, odd=0, seed=0, tensor=None, x=None):
    """The norm in f32 and in 8 bits, on rows of equal alignment, and what the definition makes of the former."""
    g = torch.Generator(device="cuda").manual_seed(seed + cols)
    if x is None:
        x = torch.randn(rows, cols, generator=g, device="cuda").to(tt(torch, xt))
    r = (torch.randn(rows, cols, generator=g, device="cuda") * 2).to(tt(torch, xt)) if residual else None
    w = torch.rand(cols, generator=g, device="cuda") + 0.5 if weight is None else weight
    b = torch.randn(cols, generator=g, device="cuda") if bias is None else bias
    stride = cols + odd
    _, full = rows_of(torch, rows, cols, torch.float32, stride, offset)
    _, codes = rows_of(torch, rows, cols, dtype(torch, yt), stride, offset)
    scale = torch.zeros(rows, device="cuda") if mode == "row" else torch.tensor([tensor or 3.0 / TOP[yt]], device="cuda")

    def norm(y, yt, **kw):
        fx.layer_norm_dev(ptr(x), ptr(y), rows, cols, xt, yt, ptr(w), ptr(b), "f32", y_stride=stride, residual_ptr=ptr(r), residual_type=xt,
                          stream=stream(torch), **kw)

    norm(full, "f32")
    norm(codes, yt, scale_ptr=ptr(scale), scale_mode=mode)
    torch.cuda.synchronize()
    want_scale = scale_of(torch, full, yt) if mode == "row" else scale
    assert torch.equal(scale.reshape(want_scale.shape), want_scale)
    want = eighths(torch, full, want_scale, yt)
    assert torch.equal(codes.float(), want.float())
    if yt == "i8":
        q, s = torch.zeros(rows, cols, dtype=torch.int8, device="cuda"), scale.clone()
        fx.i8_quantize_dev(ptr(full), rows, cols, ptr(q), ptr(s), "f32", mode, x_stride=stride, stream=stream(torch))
        torch.cuda.synchronize()
        assert torch.equal(q, codes) and torch.equal(s, scale)


@pytest.mark.parametrize("yt,mode", list(itertools.product(["i8", "e4m3"], ["row", "tensor"])))
@pytest.mark.parametrize("xt", ["f32", "bf16"])
def test_codes_are_those_of_the_f32_rows(cuda_torch, xt, yt, mode):
    for rows, cols in ((3, 64), (300, 320), (40, 1000), (700, 1024), (5, 4096), (20, 9000), (7, 20000)):
        both_ways(cuda_torch, rows, cols, xt, yt, mode)
        both_ways(cuda_torch, rows, cols - 1, xt, yt, mode)
        both_ways(cuda_torch, rows, cols, xt, yt, mode, residual=False, offset=1, odd=3)
    for rows, cols in ((20003, 64), (9001, 320), (6001, 512), (5003, 1024), (2600, 2048), (2500, 4096), (1300, 8192), (700, 16384)):
        both_ways(cuda_torch, rows, cols, xt, yt, mode)  # blocks that stay


def halves(torch, top, yt):
    """Values on and next to the middles between neighbouring 8-bit values under a row scale of top / TOP, which they do not exceed."""
    scale = torch.tensor([top], device="cuda") / torch.full((1,), TOP[yt], device="cuda")
    if yt == "i8":
        mid = torch.arange(-127, 127, device="cuda").float() + 0.5
    else:
        values = torch.arange(0, 127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn).float()
        mid = (values[1:] + values[:-1]) / 2
        mid = torch.cat((mid, -mid))
    half = mid * scale
    inf = torch.full_like(half, float("inf"))
    v = torch.cat((half, torch.nextafter(half, inf), torch.nextafter(half, -inf), half / 2, torch.tensor([top, -top, 0.0], device="cuda")))
    return torch.cat((v, torch.zeros(-v.numel() % 8, device="cuda")))


@pytest.mark.parametrize("yt,mode", list(itertools.product(["i8", "e4m3"], ["row", "tensor"])))
def test_codes_next_to_halves(cuda_torch, yt, mode):
    """A weight of zeros makes every row the bias: values on and next to halves of a step, from f32's smallest to its largest."""
    torch = cuda_torch
    for top in (127.0, 448.0, 3.7, 0.0123456, 1.1e30, 2.3e-17, 1e-19, 2.3e-26, 5e-30, 1e-36, 3.0e38):
        v = halves(torch, top, yt)
        tensor = top / TOP[yt]
        for rows in (3, 5000):
            x = torch.randn(rows, v.numel(), device="cuda").bfloat16()
            for bias in (v, v[:-1]):
                both_ways(torch, rows, bias.numel(), "bf16", yt, mode, False, torch.zeros_like(bias), bias, tensor=tensor,
                          x=x[:, :bias.numel()].contiguous())


@pytest.mark.parametrize("yt", ["i8", "e4m3"])
def test_tensor_scales_from_end_to_end(cuda_torch, yt):
    """One scale for the tensor, from below f32's normal numbers to past its reciprocals, of either sign: values far past the 8-bit
    range saturate."""
    torch = cuda_torch
    v = torch.cat([s * torch.logspace(-37, 38, 600, device="cuda") for s in (1, -1)])
    for tensor in (1e-40, 1e-37, 2e-29, 1e-21, 1e-3, 0.02, 5.0, 1e20, 9.9e36, 1.1e37, 3e38, -0.02, -1e-40):
        both_ways(torch, 3, 1200, "f32", yt, "tensor", False, torch.zeros_like(v), v, tensor=tensor)
        both_ways(torch, 3, 1199, "f32", yt, "tensor", False, torch.zeros_like(v[1:]), v[1:].contiguous(), tensor=tensor)
