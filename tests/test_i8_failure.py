"""Failure detection in the 8-bit linear kernels without a GPU fault: a layer whose codes are never brought, with a short limit
on every wait. The launch has to end by itself, with its copies and MMAs in flight waited for and its TMEM freed, the status
has to be reported once, and the next calls have to be right."""
import time

import pytest

import fenix_b200 as fx


@pytest.mark.parametrize("args", [(0, 0, 1000), (0, 4097, 1000), (0, 4, 0), (-1, 4, 1000), (999, 4, 1000)])
def test_selftest_refuses(args):
    assert fx.lib().fx_selftest_i8_wait_timeout(*args) == fx.FX_INVALID_ARGUMENT
    assert fx.lib().fx_last_error().startswith(b"fx_selftest_i8_wait_timeout: ")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 8, 20, 300, 2000, 4096])
def test_waits_that_run_out(cuda_torch, rows):
    import test_i8_gpu as base

    fx.i8_device_status(0)
    t0 = time.perf_counter()
    fx.check(fx.lib().fx_selftest_i8_wait_timeout(0, rows, 20_000_000))  # 20 ms
    assert time.perf_counter() - t0 < 10.0
    with pytest.raises(fx.FxError) as e:
        fx.i8_device_status(0)
    assert "gave up" in str(e.value)
    fx.i8_device_status(0)  # reported once
    base.run_linear(cuda_torch, rows, 300, 1024)
    base.run_linear(cuda_torch, 30, 64, 256)
    fx.i8_device_status(0)
