"""The 4-bit linear layer on rows that make its sums hard: values of one sign, inputs far above the others at weights
of zero, magnitudes at the ends of bf16's range, results held in more bits than the rows.

Tolerances count roundings; U, HALF and TINY as in test_token_gpu. Up to 8 rows no weight is rounded and a product of
a code and an input is exact: what is left is the sums in 32 bits. Within at most 128 inputs eight matrix instructions
add up, each losing at most 2^-22 of the magnitudes added so far; a scale's product and its addition to the warp's sum
follow every 2048 inputs, then at most 16 warps' sums in two chains: (32 + 2 k / 2048 + 10) U sum |w x| in all. The
result is rounded once more to y's type.
"""
import pytest
import test_token_gpu as base
from test_token_gpu import HALF, TINY, U, ptr, stream, tt, unpack

import fenix_b200 as fx

pytestmark = pytest.mark.gpu


def linear(torch, x, xt, yt, codes, scales, st, zp, group, x_scale=None):
    rows, k = x.shape
    n = codes.shape[0]
    y = torch.full((rows + 1, n), 7.0, device="cuda").to(tt(torch, yt))
    fx.w4_linear_dev(ptr(x), ptr(y), rows, n, k, group, ptr(codes), ptr(scales), ptr(zp), xt, yt, st,
                     x_scale_ptr=ptr(x_scale), x_scale_mode="tensor" if x_scale is not None else None,
                     stream=stream(torch))
    torch.cuda.synchronize()
    assert bool((y[rows].float() == 7.0).all())
    return y[:rows]


def few_rows_bound(torch, x, w, yt, want):
    k = x.shape[1]
    return (42 + 2 * k / 2048) * U * (x.abs() @ w.abs().t()) + (HALF[yt] + 4 * U) * want.abs() + TINY[yt]


def set_codes(codes, at, value):
    """The codes of inputs `at` (a list), in every output, to the outputs' values [n][len(at)]."""
    for j, i in enumerate(at):
        b, v = codes[:, i // 2], value[:, j]
        codes[:, i // 2] = (b & 0xf0 | v) if i % 2 == 0 else (b & 0x0f | v << 4)


@pytest.mark.parametrize("rows", [1, 2, 8])
@pytest.mark.parametrize("xt,yt", [("f16", "f16"), ("e4m3", "f16"), ("bf16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("kind", ["one sign", "constant", "shifted", "random"])
def test_few_rows_of_one_sign(cuda_torch, rows, xt, yt, kind):
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(rows)
    k, n = 8192, 200
    for group, zeros in ((128, False), (128, True), (64, True), (32, False)):
        codes, scales, zp = base.make_layer(torch, n, k, group, "f16", zeros, g, False)
        x = torch.randn(rows, k, generator=g, device="cuda")
        x = {"one sign": x.abs(), "constant": torch.full_like(x, 1.5), "shifted": x + 3.0, "random": x}[kind]
        x = x.to(tt(torch, xt))
        sc = torch.ones(1, device="cuda") if xt == "e4m3" else None
        y = linear(torch, x, xt, yt, codes, scales, "f16", zp, group, sc)
        xv, w = x.double(), unpack(torch, codes, scales, zp, group)
        want = xv @ w.t()
        err, lim = (y.double() - want).abs(), few_rows_bound(torch, xv, w, yt, want)
        assert bool((err <= lim).all()), ((err / lim).max().item(), group, zeros)


@pytest.mark.parametrize("rows", [1, 5, 8])
@pytest.mark.parametrize("xt,loud", [("f16", 1e4), ("f16", 6e4), ("bf16", 1e6), ("bf16", 1e12), ("e4m3", 448.0)])
@pytest.mark.parametrize("zeros", [False, True])
def test_few_rows_with_loud_inputs_at_weights_of_zero(cuda_torch, rows, xt, loud, zeros):
    """A weight whose code is its zero point is zero: however large its input, nothing of it is in the result."""
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(7)
    k, n = 2048, 150
    for group in (32, 64, 128, 256):
        codes, scales, zp = base.make_layer(torch, n, k, group, "f16", zeros, g, False)
        at = list(range(group // 3, k, group))
        zero = zp if zeros else torch.full((n, k // group), 8, dtype=torch.uint8, device="cuda")
        set_codes(codes, at, zero)
        x = torch.randn(rows, k, generator=g, device="cuda") * (0.01 if xt != "e4m3" else 0.25)
        x[:, at] = loud
        x = x.to(tt(torch, xt))
        sc = torch.ones(1, device="cuda") if xt == "e4m3" else None
        y = linear(torch, x, xt, "f16", codes, scales, "f16", zp, group, sc)
        xv, w = x.double(), unpack(torch, codes, scales, zp, group)
        want = xv @ w.t()
        err, lim = (y.double() - want).abs(), few_rows_bound(torch, xv, w, "f16", want)
        assert bool((err <= lim).all()), ((err / lim).max().item(), group)


@pytest.mark.parametrize("rows", [1, 3, 8, 9, 40])
@pytest.mark.parametrize("power", [123, 100, -90, -110])
def test_bf16_rows_at_the_ends_of_the_range(cuda_torch, rows, power):
    """Whole numbers times a power of two, with scales that bring the results back: nothing to round before the end."""
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(power + 200)
    n, k = 90, 1024
    for group, zeros in ((128, False), (64, True), (32, True)):
        codes, scales, zp = base.make_layer(torch, n, k, group, "f32", zeros, g, True)
        scales *= 2.0 ** (-power // 2)
        x = (torch.randint(-4, 5, (rows, k), generator=g, device="cuda") * 2.0 ** power).bfloat16()
        y = linear(torch, x, "bf16", "bf16", codes, scales, "f32", zp, group)
        want = x.double() @ unpack(torch, codes, scales, zp, group).t()
        assert torch.equal(y, want.float().bfloat16())


@pytest.mark.parametrize("rows", [9, 20, 128, 130, 257, 513])
@pytest.mark.parametrize("st,zeros,group", [("f16", False, 128), ("f32", True, 64), ("bf16", True, 32)])
def test_f16_results_of_many_bf16_rows(cuda_torch, rows, st, zeros, group):
    """A result held in 11 bits is not made of weights held in 8. A weight is two bf16 terms (and so is a scale of
    more bits): off by at most HALF^2 each, 2^-15 |w| together, with an input's sign, so that 4 2^-15 sqrt(sum (w x)^2)
    bounds their sum as in test_token_gpu, and one rounding to f16 remains."""
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(rows)
    worst = 0.0
    for n, k, stride, kind in ((200, 512, 0, "random"), (700, 2048, 0, "random"), (65, 1152, 1160, "one sign"),
                               (130, 512, 515, "random")):
        codes, scales, zp = base.make_layer(torch, n, k, group, st, zeros, g, False)
        _, x = base.rows_of(torch, rows, k, torch.bfloat16, stride)
        x.copy_(torch.randn(rows, k, generator=g, device="cuda"))
        if kind == "one sign":
            x.abs_()
        y = torch.empty(rows, n, dtype=torch.float16, device="cuda")
        fx.w4_linear_dev(ptr(x), ptr(y), rows, n, k, group, ptr(codes), ptr(scales), ptr(zp), "bf16", "f16", st, stride,
                         stream=stream(torch))
        torch.cuda.synchronize()
        xv, w = x.double(), unpack(torch, codes, scales, zp, group)
        want = xv @ w.t()
        lim = (4 * 2.0 ** -15 * (xv.square() @ w.square().t()).sqrt() + k / 16 * 2.0 ** -22 * (xv.abs() @ w.abs().t())
               + (HALF["f16"] + 4 * U) * want.abs() + TINY["f16"])
        err = (y.double() - want).abs()
        worst = max(worst, (err / lim).max().item())
        print(rows, st, n, k, "rms error / rms result %.2e" % (err.square().mean().sqrt() / want.square().mean().sqrt()).item())
    assert worst <= 1, worst


@pytest.mark.parametrize("rows", [9, 130, 300])
def test_two_terms_keep_what_is_not_finite_apart(cuda_torch, rows):
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(rows)
    n, k, group = 300, 512, 64
    codes, scales, zp = base.make_layer(torch, n, k, group, "f32", True, g, True)
    x = torch.randint(-4, 5, (rows, k), generator=g, device="cuda").bfloat16()
    want = (x.double() @ unpack(torch, codes, scales, zp, group).t()).half()
    x[2, 7], x[5, 100] = float("inf"), float("nan")
    scales[3, 1], scales[4, 0] = float("inf"), float("nan")
    y = linear(torch, x, "bf16", "f16", codes, scales, "f32", zp, group)
    fine_rows = [r for r in range(rows) if r not in (2, 5)]
    fine_outs = [o for o in range(n) if o not in (3, 4)]
    assert torch.equal(y[fine_rows][:, fine_outs], want[fine_rows][:, fine_outs])
    assert not bool(y[[2, 5]].isfinite().any()) and not bool(y[:, [3, 4]].isfinite().any())


def test_two_terms_captured_and_repeated(cuda_torch):
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(8)
    n, k, group = 640, 4096, 128
    codes, scales, zp = base.make_layer(torch, n, k, group, "f16", False, g, False)
    for rows in (20, 300):
        x = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
        first = linear(torch, x, "bf16", "f16", codes, scales, "f16", zp, group)
        y = torch.zeros(rows, n, dtype=torch.float16, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            fx.w4_linear_dev(ptr(x), ptr(y), rows, n, k, group, ptr(codes), ptr(scales), x_type="bf16", y_type="f16",
                             stream=stream(torch))
        for _ in range(3):
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, first)
