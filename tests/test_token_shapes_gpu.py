"""Shapes of the token-row calls that take each of the kernels' ways: tiles of 32 outputs and of 16, ranges of the
inputs times tiles, several launches, teams that walk over many rows. Inputs of the linear layers are whole numbers
times powers of two, so their results are exact and whatever is read or written in the wrong place shows; the norm's
tolerances are test_token_gpu's."""
import pytest
import test_token_gpu as base
from test_token_gpu import HALF, U, ptr, stream, tt, unpack

import fenix_b200 as fx

pytestmark = pytest.mark.gpu


# ---- the linear layer up to 8 rows: outputs past 32 a SM go in tiles of 32, the others in tiles of 16 ------------


@pytest.mark.parametrize("rows", [1, 2, 3, 8])
@pytest.mark.parametrize("xt,yt,zeros,group", [
    ("bf16", "bf16", False, 128), ("bf16", "f16", True, 64), ("f16", "f16", True, 128), ("f16", "bf16", False, 32),
    ("e4m3", "bf16", True, 64), ("e4m3", "f16", False, 32), ("bf16", "bf16", True, 32), ("e4m3", "bf16", True, 128)])
def test_few_rows_wide_tiles(cuda_torch, rows, xt, yt, zeros, group):
    sms = cuda_torch.cuda.get_device_properties(0).multi_processor_count
    for n, k, ys in ((32 * sms, 512, 0), (32 * sms + 21, 1152, 0), (3 * 32 * sms + 133, 640, 3 * 32 * sms + 150)):
        base.run_linear(cuda_torch, rows, n, k, group, xt, yt, zeros=zeros, bias=rows != 2, ys=ys)


@pytest.mark.parametrize("rows,n,k,group,xt,zeros", [
    (8, 5003, 8192, 128, "bf16", False), (8, 5003, 8192, 64, "f16", True), (5, 9600, 8192, 32, "e4m3", True),
    (8, 6000, 28672, 128, "bf16", True), (3, 4800, 28672, 256, "f16", False), (1, 5000, 57344, 32, "bf16", True),
    (8, 1000, 16384 + 32, 32, "bf16", True)])
def test_few_rows_ranges_of_inputs_times_tiles(cuda_torch, rows, n, k, group, xt, zeros):
    base.run_linear(cuda_torch, rows, n, k, group, xt, "bf16", st="f32" if rows == 1 else "f16", zeros=zeros, bias=True)


def test_few_rows_more_tiles_than_a_block_has_room_for(cuda_torch):
    """Sums of earlier ranges are kept for 16 tiles of 8 rows a block: more blocks than SMs."""
    sms = cuda_torch.cuda.get_device_properties(0).multi_processor_count
    n = 32 * sms * 16 + 32 * sms + 45
    if cuda_torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB of free device memory")
    base.run_linear(cuda_torch, 8, n, 6144, 128, zeros=True, bias=True)
    cuda_torch.cuda.empty_cache()


@pytest.mark.parametrize("rows", [1, 7, 12, 200])
@pytest.mark.parametrize("st,s_off,z_off,k,group", [("f16", 1, 1, 1024, 32), ("f16", 2, 4, 4096, 32), ("f16", 0, 3, 1088, 64),
                                                    ("bf16", 3, 0, 2048, 128), ("f32", 1, 2, 992, 32), ("f16", 8, 16, 4096, 32)])
def test_scales_and_zero_points_of_any_alignment(cuda_torch, rows, st, s_off, z_off, k, group):
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(rows + k)
    for n in (333, 5000):
        codes, scales, zp = base.make_layer(torch, n, k, group, st, True, g, True)
        s = torch.full((scales.numel() + s_off + 8,), float("nan"), dtype=scales.dtype, device="cuda")
        z = torch.full((zp.numel() + z_off + 16,), 255, dtype=torch.uint8, device="cuda")
        s[s_off:s_off + scales.numel()] = scales.flatten()
        z[z_off:z_off + zp.numel()] = zp.flatten()
        x = torch.randint(-4, 5, (rows, k), generator=g, device="cuda").bfloat16()
        y = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
        fx.w4_linear_dev(ptr(x), ptr(y), rows, n, k, group, ptr(codes), s.data_ptr() + s_off * s.element_size(),
                         z.data_ptr() + z_off, scale_type=st, stream=stream(torch))
        torch.cuda.synchronize()
        want = x.double() @ unpack(torch, codes, scales, zp, group).t()
        assert torch.equal(y, want.float().bfloat16()), n


# ---- several launches of a call ---------------------------------------------------------------------------------


@pytest.mark.parametrize("xt", ["bf16", "e4m3"])
def test_linear_rows_of_two_launches(cuda_torch, xt):
    base.run_linear(cuda_torch, 65535 * 16 + 17, 16, 32, 32, xt, "bf16", zeros=True, bias=True)
    cuda_torch.cuda.empty_cache()


@pytest.mark.parametrize("ot", ["f32", "bf16"])
def test_dequantize_outputs_of_two_launches(cuda_torch, ot):
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(2)
    n, k = 65535 + 3, 32
    codes, scales, zp = base.make_layer(torch, n, k, 32, "f16", True, g, True)
    out = torch.full((n + 1, k), 7.0, device="cuda").to(tt(torch, ot))
    fx.w4_dequantize_dev(ptr(codes), ptr(scales), n, k, 32, ptr(out), ptr(zp), ot, "f16", stream=stream(torch))
    torch.cuda.synchronize()
    assert torch.equal(out[:n].double(), unpack(torch, codes, scales, zp, 32)) and bool((out[n].float() == 7.0).all())


# ---- norm: every team, over at least three rows a block ------------------------------------------------------------


@pytest.mark.parametrize("cols", [8, 64, 72, 128, 136, 256, 264, 320, 328, 512, 520, 1024, 1032, 2048, 2056, 4096, 4104, 5120,
                                  5128, 6144, 6152, 8192, 8200, 16384])
@pytest.mark.parametrize("xt,yt,residual", [("bf16", "e4m3", True), ("f16", "f16", False)])
def test_norm_teams_that_walk(cuda_torch, cols, xt, yt, residual):
    torch = cuda_torch
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    threads = 128 if cols <= 1024 else (cols + 15) // 16
    rows = 3 * sms * (2048 // threads) * (1 if cols > 1024 else max(1, 1024 // cols)) + 5
    base.run_norm(torch, rows, cols, xt, yt, xt, xt, "row" if yt == "e4m3" else None, residual, residual, seed=cols)


@pytest.mark.parametrize("cols", [320, 1000, 1024, 4096])
def test_norm_teams_that_walk_in_place(cuda_torch, cols):
    torch = cuda_torch
    rows = 3 * 148 * 16 * (2 if cols <= 1024 else 1) + 3
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(rows, cols, generator=g, device="cuda").bfloat16()
    r = torch.randn(rows, cols, generator=g, device="cuda").bfloat16()
    h, v = base.norm_want(torch, x, r, None, 1e-6)
    x1, r1, x2, y2 = x.clone(), r.clone(), x.clone(), torch.empty_like(x)
    fx.rms_norm_dev(ptr(x1), ptr(x1), rows, cols, residual_ptr=ptr(r1), sum_ptr=ptr(r1), stream=stream(torch))
    fx.rms_norm_dev(ptr(x2), ptr(y2), rows, cols, residual_ptr=ptr(r), sum_ptr=ptr(x2), stream=stream(torch))
    torch.cuda.synchronize()
    base.check_close(torch, x1, v, HALF["bf16"] + base.NORM_TOL, 0)
    base.check_close(torch, r1, h, HALF["bf16"] + 2 * U, base.TINY["bf16"])
    assert torch.equal(x2, r1) and torch.equal(y2, x1)


@pytest.mark.parametrize("cols", [200, 500, 777, 1000, 1023])
@pytest.mark.parametrize("xt", ["f32", "bf16"])
def test_norm_many_rows_that_no_team_walks_over(cuda_torch, cols, xt):
    """32-bit rows, and rows that are not aligned: a warp or a block a row."""
    base.run_norm(cuda_torch, 2500, cols, xt, "e4m3", "f32", "f32", "row", strides=(cols + 1, 0, 0, 0), seed=cols)
    base.run_norm(cuda_torch, 2500, cols // 8 * 8, "f32", "bf16", "bf16", "f32", seed=cols)


@pytest.mark.parametrize("cols", [16392, 24576, 32768, 32767])
@pytest.mark.parametrize("xt", ["f32", "bf16"])
def test_norm_longest_rows(cuda_torch, cols, xt):
    base.run_norm(cuda_torch, 500, cols, xt, "e4m3", xt, xt, "row", seed=cols)


# ---- inputs past 2^21, where a group's number no longer comes from a product ---------------------------------------


@pytest.mark.parametrize("rows", [1, 8, 12])
@pytest.mark.parametrize("group", [96, 32])
def test_inputs_past_two_million(cuda_torch, rows, group):
    k = (1 << 21) // group * group + 5 * group
    base.run_linear(cuda_torch, rows, 37, k, group, "bf16" if rows != 8 else "e4m3", "bf16", zeros=True, bias=True)
    cuda_torch.cuda.empty_cache()


def test_quantize_rows_past_two_million(cuda_torch):
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(3)
    k = 96 * 21900
    w = torch.randn(3, k, generator=g, device="cuda").bfloat16()
    codes, scales, zp = base.quantize(torch, w, "bf16", 96, "f16", True)
    want = base.quantize_want(torch, w, 96, "f16", True)
    assert torch.equal(codes, want[0]) and torch.equal(scales.float(), want[1]) and torch.equal(zp, want[2])
    out = torch.empty(3, k, device="cuda")
    fx.w4_dequantize_dev(ptr(codes), ptr(scales), 3, k, 96, ptr(out), ptr(zp), "f32", "f16", stream=stream(torch))
    assert torch.equal(out.double(), unpack(torch, codes, scales, zp, 96))
