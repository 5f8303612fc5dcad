"""The 8-bit linear layer's clusters beside kernels of another library that hold tensor memory of their own, on other streams and on its own."""
import pytest

import fenix_b200 as fx
from test_i8_gpu import linear_want
from test_token_gpu import ptr, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("captured", [False, True])
def test_linear_beside_another_librarys_products(cuda_torch, captured):
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(0)
    calls = []
    for rows, n, k in ((1, 4096, 4096), (17, 1000, 8192), (64, 2000, 4096), (128, 1500, 2048), (200, 700, 8192), (1000, 3000, 1024)):
        x = torch.randint(-127, 128, (rows, k), generator=g, device="cuda", dtype=torch.int8)
        w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
        xs, ws = torch.rand(rows, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda")
        calls.append((x, w, xs, ws, torch.empty(rows, n, device="cuda"), linear_want(torch, x, xs, w, ws, None, "f32")))
    products = []
    for rows, n, k in ((64, 512, 1024), (300, 1000, 512), (2048, 2048, 1024), (16, 4096, 4096)):
        a = torch.randint(-3, 4, (rows, k), generator=g, device="cuda").bfloat16()
        b = torch.randint(-3, 4, (k, n), generator=g, device="cuda").bfloat16()
        products.append((a, b, torch.empty(rows, n, dtype=torch.bfloat16, device="cuda"), (a.double() @ b.double()).bfloat16()))

    def ours():
        for x, w, xs, ws, y, _ in calls:
            fx.i8_linear_dev(ptr(x), ptr(y), *y.shape, x.shape[1], ptr(w), ptr(ws), ptr(xs), "f32", stream=stream(torch))

    def theirs():
        for a, b, out, _ in products:
            torch.mm(a, b, out=out)

    def turns():  # on one stream, one after the other
        for (x, w, xs, ws, y, _), (a, b, out, _) in zip(calls * 2, products * 3):
            torch.mm(a, b, out=out)
            fx.i8_linear_dev(ptr(x), ptr(y), *y.shape, x.shape[1], ptr(w), ptr(ws), ptr(xs), "f32", stream=stream(torch))

    streams = [torch.cuda.Stream() for _ in range(3)]
    run = []
    for on, call in zip(streams, (ours, theirs, turns)):
        with torch.cuda.stream(on):
            call()  # the library's own preparations
        torch.cuda.synchronize()
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=on):
                call()
            call = graph.replay
        run.append((on, call))
    for call in calls:
        call[4].fill_(-1.0)
    torch.cuda.synchronize()
    for _ in range(20):
        for on, call in run:
            with torch.cuda.stream(on):
                call()
    torch.cuda.synchronize()
    for *_, y, want in calls:
        assert torch.equal(y, want)
    for *_, out, want in products:
        assert torch.equal(out, want)  # whole numbers below 2^24
    fx.i8_device_status(0)
