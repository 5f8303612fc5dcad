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


FIRST = """
import sys
sys.path[:0] = ["tests", "."]
import torch
import fenix_b200 as fx
from test_i8_gpu import linear_want
from test_token_gpu import ptr, stream

g = torch.Generator(device="cuda").manual_seed(0)
calls = []
for rows, n, k in ((8, 4096, 2048), (100, 2000, 4096), (300, 512, 8192), (1000, 3000, 1024), (5, 700, 999)):
    x = torch.randint(-127, 128, (rows, k), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    xs, ws, y = torch.rand(rows, device="cuda"), torch.rand(n, device="cuda"), torch.zeros(rows, n, device="cuda")
    calls.append((rows, n, k, x, w, xs, ws, y))
h = torch.randn(3000, 1024, device="cuda").bfloat16()
out, dx = torch.zeros_like(h), torch.zeros_like(h)
mean, rstd = torch.zeros(3000, device="cuda"), torch.zeros(3000, device="cuda")
dw, db = torch.zeros(1024, device="cuda"), torch.zeros(1024, device="cuda")
work = torch.empty(fx.layer_norm_backward_workspace(3000, 1024), dtype=torch.uint8, device="cuda")
codes, scale = torch.zeros(3000, 1024, dtype=torch.int8, device="cuda"), torch.zeros(3000, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    for rows, n, k, x, w, xs, ws, y in calls:
        fx.i8_linear_dev(ptr(x), ptr(y), rows, n, k, ptr(w), ptr(ws), ptr(xs), "f32", stream=stream(torch))
    fx.layer_norm_dev(ptr(h), ptr(out), 3000, 1024, mean_ptr=ptr(mean), rstd_ptr=ptr(rstd), stream=stream(torch))
    fx.layer_norm_backward_dev(ptr(h), ptr(h), ptr(mean), ptr(rstd), 3000, 1024, dx_ptr=ptr(dx), dweight_ptr=ptr(dw), dbias_ptr=ptr(db),
                               work_ptr=ptr(work), work_bytes=work.numel(), stream=stream(torch))
    fx.i8_quantize_dev(ptr(h), 3000, 1024, ptr(codes), ptr(scale), stream=stream(torch))
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
for rows, n, k, x, w, xs, ws, y in calls:
    assert torch.equal(y, linear_want(torch, x, xs, w, ws, None, "f32")), (rows, n, k)
once = [t.clone() for t in (out, mean, rstd, dx, dw, db, codes, scale)]
fx.layer_norm_dev(ptr(h), ptr(out), 3000, 1024, mean_ptr=ptr(mean), rstd_ptr=ptr(rstd), stream=stream(torch))
fx.layer_norm_backward_dev(ptr(h), ptr(h), ptr(mean), ptr(rstd), 3000, 1024, dx_ptr=ptr(dx), dweight_ptr=ptr(dw), dbias_ptr=ptr(db),
                           work_ptr=ptr(work), work_bytes=work.numel(), stream=stream(torch))
fx.i8_quantize_dev(ptr(h), 3000, 1024, ptr(codes), ptr(scale), stream=stream(torch))
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(once, (out, mean, rstd, dx, dw, db, codes, scale)))
assert bool(scale.gt(0).all()) and bool(dx.isfinite().all())
print("captured")
"""


@pytest.mark.gpu
def test_first_calls_of_a_process_are_captured(cuda_torch, root):
    import subprocess
    import sys

    done = subprocess.run([sys.executable, "-c", FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]
