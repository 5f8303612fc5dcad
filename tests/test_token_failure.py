"""Failure detection in the 4-bit linear kernels without a GPU fault: a layer whose codes are never brought, with a
short limit on every wait. The launch has to end by itself, with its copies and MMAs in flight waited for and its
TMEM freed, the status has to be reported once, and the next calls have to be right."""
import time

import pytest

import fenix_b200 as fx

F32, F16, BF16, E4M3 = 0, 1, 2, 3


@pytest.mark.parametrize("args", [(0, F32, 4, 1000), (0, 7, 4, 1000), (0, BF16, 0, 1000), (0, BF16, 4097, 1000),
                                  (0, BF16, 4, 0), (-1, BF16, 4, 1000), (999, BF16, 4, 1000)])
def test_selftest_refuses(args):
    assert fx.lib().fx_selftest_w4_wait_timeout(*args) == fx.FX_INVALID_ARGUMENT
    assert fx.lib().fx_last_error().startswith(b"fx_selftest_w4_wait_timeout: ")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 8, 20, 300, 2000])
@pytest.mark.parametrize("xt", ["bf16", "f16", "e4m3"])
def test_waits_that_run_out(cuda_torch, rows, xt):
    import test_token_gpu as base

    fx.w4_device_status(0)
    t0 = time.perf_counter()
    fx.check(fx.lib().fx_selftest_w4_wait_timeout(0, fx.DTYPES[xt], rows, 20_000_000))  # 20 ms
    assert time.perf_counter() - t0 < 10.0
    with pytest.raises(fx.FxError) as e:
        fx.w4_device_status(0)
    assert "gave up" in str(e.value)
    fx.w4_device_status(0)  # reported once
    base.run_linear(cuda_torch, rows, 300, 1024, 128, xt)
    base.run_linear(cuda_torch, 30, 64, 256, 64)
    fx.w4_device_status(0)
