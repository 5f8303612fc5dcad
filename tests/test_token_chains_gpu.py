"""Chains of calls that work in place, on rows that share cache lines with their neighbours: every call sees all that the one before it wrote,
though it begins while that one ends. Each is compared bit for bit with the same calls one at a time."""
import pytest

import fenix_b200 as fx
from test_token_gpu import ptr, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(7, 77), (3000, 77), (5000, 333), (3000, 1001), (2000, 2049), (1500, 5119), (700, 9999), (400, 20001)])
@pytest.mark.parametrize("captured", [False, True])
def test_norms_in_place(cuda_torch, rows, cols, captured):
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(cols)
    start = torch.randn(rows, cols, generator=g, device="cuda").bfloat16()
    weight = (torch.rand(cols, generator=g, device="cuda") * 2).bfloat16()
    bias = torch.randn(cols, generator=g, device="cuda").bfloat16()
    work = torch.empty(fx.layer_norm_backward_workspace(rows, cols), dtype=torch.uint8, device="cuda")

    class State:
        def __init__(self):
            self.x, self.dx = start.clone(), start.clone()
            self.q, self.qs = torch.zeros(rows, cols, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
            self.mean, self.rstd = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
            self.dw, self.db = torch.zeros(cols, device="cuda"), torch.zeros(cols, device="cuda")

        def all(self):
            return self.x, self.dx, self.q, self.qs, self.mean, self.rstd, self.dw, self.db

        def steps(self):
            st = stream(torch)
            x, q, qs, mean, rstd = (ptr(t) for t in (self.x, self.q, self.qs, self.mean, self.rstd))
            for _ in range(6):
                yield fx.layer_norm_dev(x, x, rows, cols, weight_ptr=ptr(weight), bias_ptr=ptr(bias), mean_ptr=mean, rstd_ptr=rstd, stream=st)
                yield fx.layer_norm_dev(x, x, rows, cols, weight_ptr=ptr(bias), mean_ptr=mean, rstd_ptr=rstd, stream=st)
                yield fx.i8_quantize_dev(x, rows, cols, q, qs, stream=st)
                yield fx.i8_dequantize_dev(q, qs, rows, cols, x, stream=st)
                yield fx.layer_norm_backward_dev(ptr(self.dx), x, mean, rstd, rows, cols, weight_ptr=ptr(weight), dsum_ptr=x, dx_ptr=ptr(self.dx),
                                                 dweight_ptr=ptr(self.dw), dbias_ptr=ptr(self.db), accumulate=True, work_ptr=ptr(work),
                                                 work_bytes=work.numel(), stream=st)
                yield fx.layer_norm_dev(ptr(self.dx), ptr(self.dx), rows, cols, stream=st)

    one = State()
    for _ in one.steps():
        torch.cuda.synchronize()
    assert all(bool(t.float().isfinite().all()) for t in one.all()) and bool(one.x.any()) and bool(one.dx.any())
    states = [State() for _ in range(8)]
    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for s in states:
                for _ in s.steps():
                    pass
        graph.replay()
    else:
        for s in states:
            for _ in s.steps():
                pass
    torch.cuda.synchronize()
    for s in states:
        assert all(torch.equal(p, q) for p, q in zip(s.all(), one.all()))
