"""Shapes of the token-row calls that take each of the kernels' ways: tiles of 32 outputs and of 16, ranges of the
inputs times tiles, several launches, teams that walk over many rows. Inputs of the linear layers are whole numbers
times powers of two, so their results are exact and whatever is read or written in the wrong place shows; the norm's
tolerances are test_token_gpu's."""
import pytest
import test_token_gpu as base
from test_token_gpu import ptr, stream, unpack

import fenix_b200 as fx

pytestmark = pytest.mark.gpu


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
