"""The 8-bit integer linear layer and its quantiser on the GPU against plain implementations in 64 bits.

Sums of products of two bytes are whole numbers below 2^31: f64 holds them exactly, and the three operations in f32 after
them (times the token's scale, times the channel's, plus the bias) round once each, as torch's do on the same f32 values.
So results are compared bit for bit, save where a test says otherwise."""
import itertools

import pytest

import fenix_b200 as fx
from test_token_gpu import HALF, TINY, U, check_close, ptr, rows_of, stream, tt

pytestmark = pytest.mark.gpu


# ---- quantiser --------------------------------------------------------------------------------------------------


def quantize_want(torch, x, scale=None):
    """(codes, scales [rows, 1] or [1]) of the definition, in f32's correctly rounded quotients."""
    f = x.float()
    if scale is None:
        scale = f.abs().amax(1, keepdim=True).clamp(min=1e-30) / torch.full((1,), 127.0, device=x.device)
    return torch.round(f / scale).clamp(-127, 127).to(torch.int8), scale


def run_quantize(torch, rows, cols, xt="bf16", mode="row", xs=0, cs=0, offset=0, c_offset=0, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    _, x = rows_of(torch, rows, cols, tt(torch, xt), xs, offset)
    x.copy_(torch.randn(rows, cols, generator=g, device="cuda") * spread)
    if rows > 2:
        x[1] = 0.0
    cbuf, codes = rows_of(torch, rows, cols, torch.int8, cs, c_offset, 99)
    scale = torch.full((rows + 1,), 5.0, device="cuda") if mode == "row" else torch.tensor([0.02 * spread], device="cuda")
    fx.i8_quantize_dev(ptr(x), rows, cols, ptr(codes), ptr(scale), xt, mode, xs, cs, stream(torch))
    torch.cuda.synchronize()
    want, sc = quantize_want(torch, x, None if mode == "row" else scale)
    assert torch.equal(codes, want)
    if mode == "row":
        assert torch.equal(scale[:rows, None], sc) and scale[rows].item() == 5.0
    for yt in ("f32", "f16", "bf16"):
        ybuf, y = rows_of(torch, rows, cols, tt(torch, yt), xs, offset, 7.0)
        fx.i8_dequantize_dev(ptr(codes), ptr(scale), rows, cols, ptr(y), yt, mode, cs, xs, stream(torch))
        torch.cuda.synchronize()
        assert torch.equal(y, (want.float() * sc).to(y.dtype))
        y.fill_(7.0)
        assert bool((ybuf == 7.0).all())
    codes.fill_(99)
    assert bool((cbuf == 99).all())


@pytest.mark.parametrize("cols", [1, 2, 7, 8, 31, 64, 65, 72, 100, 256, 264, 511, 512, 520, 1000, 1024, 1032, 2048, 2056, 4095,
                                  4096, 4104, 8192, 8200, 16384, 16392, 16385, 40000, 131071])
@pytest.mark.parametrize("rows", [1, 3, 130])
def test_quantize_extents(cuda_torch, rows, cols):
    run_quantize(cuda_torch, rows, cols, "bf16", seed=cols)
    run_quantize(cuda_torch, rows, cols, "f32", "tensor", cs=(cols + 15) // 16 * 16, seed=cols + 1)


@pytest.mark.parametrize("xt,mode", list(itertools.product(["f32", "f16", "bf16"], ["row", "tensor"])))
def test_quantize_types_strides_and_offsets(cuda_torch, xt, mode):
    for xs, cs, offset, c_offset in ((0, 0, 0, 0), (336, 336, 8, 16), (331, 0, 1, 0), (0, 333, 0, 3), (340, 340, 4, 4)):
        for cols in (328, 330):
            run_quantize(cuda_torch, 37, cols, xt, mode, max(xs, cols) if xs else 0, max(cs, cols) if cs else 0, offset, c_offset,
                         seed=cols)
    for spread in (1e-3, 1e3):
        run_quantize(cuda_torch, 50, 4096, xt, mode, spread=spread)


def test_quantize_many_rows(cuda_torch):
    run_quantize(cuda_torch, 200001, 8, "f16")
    run_quantize(cuda_torch, 70001, 136, "bf16", "tensor")


def test_quantize_rounds_the_quotient(cuda_torch):
    """Values on and next to halves of a step, where a product with the reciprocal would round the other way now and then."""
    torch = cuda_torch
    for top in (127.0, 3.7, 0.0123456, 1.1e30, 2.3e-20, 3.0e38):
        scale = torch.tensor([top], device="cuda") / torch.tensor([127.0], device="cuda")
        half = (torch.arange(-127, 127, device="cuda").float() + 0.5) * scale
        up = torch.nextafter(half, torch.full_like(half, float("inf")))
        down = torch.nextafter(half, torch.full_like(half, -float("inf")))
        x = torch.cat((half, up, down, torch.tensor([top, -top], device="cuda"))).reshape(1, -1).repeat(3, 1).contiguous()
        codes = torch.empty(3, x.shape[1], dtype=torch.int8, device="cuda")
        got = torch.empty(3, device="cuda")
        fx.i8_quantize_dev(ptr(x), 3, x.shape[1], ptr(codes), ptr(got), "f32", stream=stream(torch))
        want, sc = quantize_want(torch, x)
        assert torch.equal(got[:, None], sc) and torch.equal(codes, want)


@pytest.mark.parametrize("cols", [40, 77, 4096, 20000])
def test_quantize_extreme_rows(cuda_torch, cols):
    torch = cuda_torch
    inf, nan = float("inf"), float("nan")
    x = torch.randn(8, cols, device="cuda")
    x[0, 3], x[1, 4], x[2, 5] = nan, inf, -inf
    x[3] *= 1e-38   # subnormal quotients' scale: the floor
    x[4] = 3.0e38
    x[5] = 0.0
    x[6] = 1e-30
    codes = torch.empty(8, cols, dtype=torch.int8, device="cuda")
    scale = torch.empty(8, device="cuda")
    fx.i8_quantize_dev(ptr(x), 8, cols, ptr(codes), ptr(scale), "f32", stream=stream(torch))
    torch.cuda.synchronize()
    assert bool(scale[0].isnan()) and bool((scale[1:3] == inf).all()) and bool((codes[:3] == 0).all())
    want, sc = quantize_want(torch, x[3:])
    assert torch.equal(codes[3:], want) and torch.equal(scale[3:, None], sc)
    one = torch.tensor([0.01], device="cuda")
    fx.i8_quantize_dev(ptr(x), 8, cols, ptr(codes), ptr(one), "f32", "tensor", stream=stream(torch))
    torch.cuda.synchronize()
    want = torch.round(x.nan_to_num(0.0, inf, -inf) / one).clamp(-127, 127).to(torch.int8)
    assert torch.equal(codes, want)
    for tiny in (1e-40, 2.0e38):  # a reciprocal past f32's range, and one below its normal numbers
        one.fill_(tiny)
        fx.i8_quantize_dev(ptr(x), 8, cols, ptr(codes), ptr(one), "f32", "tensor", stream=stream(torch))
        torch.cuda.synchronize()
        assert torch.equal(codes, torch.round(x.nan_to_num(0.0, inf, -inf) / one).clamp(-127, 127).to(torch.int8))


def test_quantize_past_32_bits(cuda_torch):
    torch = cuda_torch
    rows, cols, stride = 1100, 64, 1 << 22
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    run_quantize(torch, rows, cols, "bf16", xs=stride)
    torch.cuda.empty_cache()
    run_quantize(torch, rows, cols, "bf16", cs=stride)
    torch.cuda.empty_cache()


# ---- linear -----------------------------------------------------------------------------------------------------


def linear_want(torch, x, x_scale, codes, scales, bias, yt):
    s = (x.double() @ codes.double().t()).float()  # exact in f64, one rounding to f32
    y = s * x_scale.reshape(-1, 1) * scales
    if bias is not None:
        y = y + bias
    return y.to(tt(torch, yt))


def run_linear(torch, rows, n, k, yt="bf16", mode="row", bias=False, xs=0, ws=0, ys=0, offset=0, w_offset=0, y_offset=0, seed=0,
               low=-128, high=128, scale=None):
    """Rows 16-byte aligned unless strides or offsets say otherwise: xs and ws 0 are k rounded up to 16."""
    g = torch.Generator(device="cuda").manual_seed(seed + rows + n + k)
    xs, ws = xs or (k + 15) // 16 * 16, ws or (k + 15) // 16 * 16
    xbuf, x = rows_of(torch, rows, k, torch.int8, xs, offset, 77)  # what lies between the rows must not be multiplied
    wbuf, w = rows_of(torch, n, k, torch.int8, ws, w_offset, -77)
    x.copy_(torch.randint(low, high, (rows, k), generator=g, device="cuda", dtype=torch.int8))
    w.copy_(torch.randint(low, high, (n, k), generator=g, device="cuda", dtype=torch.int8))
    size = scale or 1.0 / (64 * k ** 0.5)
    x_scale = (torch.rand(rows if mode == "row" else 1, generator=g, device="cuda") + 0.5) * size
    scales = (torch.rand(n, generator=g, device="cuda") + 0.5) * (1 / 64)
    b = torch.randn(n, generator=g, device="cuda") if bias else None
    ybuf, y = rows_of(torch, rows, n, tt(torch, yt), ys, y_offset, 7.0)
    fx.i8_linear_dev(ptr(x), ptr(y), rows, n, k, ptr(w), ptr(scales), ptr(x_scale), yt, mode, xs, ys, ws, ptr(b), stream(torch))
    torch.cuda.synchronize()
    want = linear_want(torch, x, x_scale, w, scales, b, yt)
    assert torch.equal(y, want), (y.double() - want.double()).abs().max().item()
    y.fill_(7.0)
    assert bool((ybuf == 7.0).all())  # nothing outside the rows was written


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 48, 64, 65, 100, 128, 129, 160, 192, 200, 255, 256, 257,
                                  300, 384, 500, 512, 513, 777, 1000])
def test_linear_rows(cuda_torch, rows):
    run_linear(cuda_torch, rows, 300, 512)
    run_linear(cuda_torch, rows, 131, 208, "f16", bias=True)
    run_linear(cuda_torch, rows, 1000, 1040, "f32", "tensor")


@pytest.mark.parametrize("n", [1, 2, 7, 8, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 255, 256, 257, 511, 777, 4096, 5003])
def test_linear_outputs(cuda_torch, n):
    for rows in (1, 5, 20, 70, 300):
        run_linear(cuda_torch, rows, n, 256, "bf16", bias=n % 2 == 1)


@pytest.mark.parametrize("k", [1, 2, 3, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 144, 255, 256, 257, 500, 512, 1000, 1024,
                               1025, 2047, 4096, 4705, 8192, 16384, 20000])
def test_linear_inner(cuda_torch, k):
    for rows in (1, 6, 33, 140, 600):
        run_linear(cuda_torch, rows, 200, k, "f16", bias=True)


@pytest.mark.parametrize("yt,mode,bias", list(itertools.product(["f32", "f16", "bf16"], ["row", "tensor"], [False, True])))
def test_linear_types(cuda_torch, yt, mode, bias):
    for rows in (1, 4, 17, 150, 400):
        run_linear(cuda_torch, rows, 264, 384, yt, mode, bias)
        run_linear(cuda_torch, rows, 259, 390, yt, mode, bias)


@pytest.mark.parametrize("xs,ws,ys,offset,w_offset,y_offset", [
    (512, 528, 264, 16, 32, 8), (501, 0, 0, 0, 0, 0), (0, 503, 0, 0, 0, 0), (0, 0, 251, 0, 0, 0), (0, 0, 0, 1, 0, 0),
    (0, 0, 0, 0, 5, 0), (0, 0, 0, 0, 0, 1), (0, 0, 256, 0, 0, 4), (504, 508, 252, 4, 8, 2), (501, 502, 253, 3, 7, 5)])
def test_linear_strides_and_offsets(cuda_torch, xs, ws, ys, offset, w_offset, y_offset):
    for rows, k in itertools.product((1, 6, 20, 130, 300), (500, 481)):
        for yt in ("bf16", "f32"):
            run_linear(cuda_torch, rows, 250, k, yt, "row", True, xs, ws, ys, offset, w_offset, y_offset)


def test_linear_sums_at_the_border(cuda_torch):
    """-128 times -128, as many times as 32 bits hold: no sum wraps, none is held in fewer bits."""
    for rows in (1, 8, 20, 300):
        run_linear(cuda_torch, rows, 130, 131071, "f32", low=-128, high=-127, scale=2.0 ** -20)
        run_linear(cuda_torch, rows, 130, 131071, "f32", low=126, high=128, scale=2.0 ** -20)


def test_linear_large(cuda_torch):
    run_linear(cuda_torch, 1, 28672, 8192, "f16")
    run_linear(cuda_torch, 8, 14336, 4096)
    run_linear(cuda_torch, 2000, 1500, 4096)
    run_linear(cuda_torch, 1500, 3000, 2048, "f16", bias=True)
    run_linear(cuda_torch, 5000, 4100, 1024, "f32")


@pytest.mark.parametrize("tiles", [9, 15, 16, 18, 19, 22, 23, 33, 37, 45, 46, 74, 75, 148, 149])
def test_linear_ranges_of_inputs(cuda_torch, tiles):
    """Tiles of 128 outputs whose inputs are cut into ranges, as many as the GPU has room for; the last tile is a part."""
    run_linear(cuda_torch, 20, tiles * 128 - 5, 3584, bias=True)
    run_linear(cuda_torch, 3, tiles * 128 - 64, 2176 + 16)
    run_linear(cuda_torch, 130, tiles * 128, 1000, "f16")


@pytest.mark.parametrize("rows,n", [(2005, 5003), (1003, 9001), (4096, 2000), (513, 20000)])
def test_linear_tiles_that_fill_the_gpu(cuda_torch, rows, n):
    run_linear(cuda_torch, rows, n, 1120, bias=True)
    run_linear(cuda_torch, rows, n, 999, "f16", ys=n + 5)


@pytest.mark.parametrize("rows", [33, 48, 100, 127, 128])
def test_linear_few_rows_of_wide_layers(cuda_torch, rows):
    """Fewer rows than half a pair's tile, past more outputs than the stream takes."""
    run_linear(cuda_torch, rows, 10000, 272, bias=True)
    run_linear(cuda_torch, rows, 9479, 1000, "f16", "tensor")
    run_linear(cuda_torch, rows, 9601, 130, "f32", y_offset=1)


@pytest.mark.parametrize("rows", [129, 200, 256, 300, 512, 600])
@pytest.mark.parametrize("n,k", [(256, 16384), (1000, 8192), (77, 5000), (4096, 4096), (5003, 2000), (2500, 3000), (640, 9300)])
def test_linear_clusters_of_pairs(cuda_torch, rows, n, k):
    """Few tiles of many inputs, which two to four pairs share; the last range may be a part, results aligned or not."""
    run_linear(cuda_torch, rows, n, k)
    run_linear(cuda_torch, rows, n, k, "f32", bias=True)
    run_linear(cuda_torch, rows, n, k, "f16", "tensor", ys=n + 5, y_offset=3)


def test_linear_kernels_of_all_kinds_at_once(cuda_torch):
    """Calls that take different kernels, with and without tensor memory of their own, on streams of their own at once."""
    torch = cuda_torch
    g = torch.Generator(device="cuda").manual_seed(4)
    calls = []
    for rows, n, k, pitch in ((1, 4096, 2048, 2048), (60, 2000, 4096, 4096), (100, 1500, 1024, 1024), (100, 12000, 512, 512),
                              (300, 700, 8192, 8192), (1000, 2100, 1024, 1024), (70, 300, 999, 999)):
        x = torch.randint(-127, 128, (rows, pitch), generator=g, device="cuda", dtype=torch.int8)
        w = torch.randint(-127, 128, (n, pitch), generator=g, device="cuda", dtype=torch.int8)
        xs, ws = torch.rand(rows, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda")
        y = torch.empty(rows, n, device="cuda")
        calls.append((torch.cuda.Stream(), y, linear_want(torch, x[:, :k], xs, w[:, :k], ws, None, "f32"),
                      lambda x=x, w=w, xs=xs, ws=ws, y=y, rows=rows, n=n, k=k: fx.i8_linear_dev(
                          ptr(x), ptr(y), rows, n, k, ptr(w), ptr(ws), ptr(xs), "f32", stream=stream(torch))))
    torch.cuda.synchronize()
    for _ in range(20):
        for on, y, _, call in calls:
            with torch.cuda.stream(on):
                y.fill_(-1.0)
                call()
    torch.cuda.synchronize()
    for _, y, want, _ in calls:
        assert torch.equal(y, want)
    fx.i8_device_status(0)


def test_linear_many_rows(cuda_torch):
    run_linear(cuda_torch, 300001, 24, 64)
    run_linear(cuda_torch, 70001, 130, 33, "f16", xs=33, ws=33)


def test_linear_rows_of_two_launches(cuda_torch):
    """More rows than one launch's second grid dimension holds in tiles of 64."""
    run_linear(cuda_torch, 65535 * 64 + 70, 3, 17, "bf16", xs=17, ws=17)
    run_linear(cuda_torch, 65535 * 64 + 70, 3, 17, "bf16")


def test_linear_past_32_bits(cuda_torch):
    torch = cuda_torch
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    for kw in (dict(xs=1 << 22), dict(ys=1 << 22), dict(xs=(1 << 22) + 1)):
        run_linear(torch, 1100, 128, 128, **kw)
        torch.cuda.empty_cache()
    run_linear(torch, 5, 1100, 128, ws=1 << 22)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows", [1, 5, 40, 400])
def test_linear_values_not_finite_stay_apart(cuda_torch, rows):
    """Scales that are NaN or infinite reach their own row and their own output; rows and outputs behind the last are not read."""
    torch = cuda_torch
    n, k = 200, 256
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randint(1, 5, (rows, k), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(1, 5, (n, k), generator=g, device="cuda", dtype=torch.int8)
    xs, ws = torch.ones(rows + 1, device="cuda"), torch.full((n + 1,), 2.0 ** -7, device="cuda")
    xs[rows], ws[n] = float("nan"), float("nan")
    clean = linear_want(torch, x, xs[:rows], w, ws[:n], None, "bf16")
    if rows > 1:
        xs[1] = float("nan")
    ws[3], ws[4] = float("inf"), float("nan")
    y = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    fx.i8_linear_dev(ptr(x), ptr(y), rows, n, k, ptr(w), ptr(ws), ptr(xs), stream=stream(torch))
    torch.cuda.synchronize()
    keep = [i for i in range(rows) if i != 1]
    others = [i for i in range(n) if i not in (3, 4)]
    assert torch.equal(y[keep][:, others], clean[keep][:, others])
    assert bool((y[keep, 3] == float("inf")).all()) and bool(y[:, 4].isnan().all())
    assert rows == 1 or bool(y[1].isnan().all())


def test_linear_a_row_does_not_depend_on_the_others(cuda_torch):
    torch = cuda_torch
    n, k = 700, 1500
    g = torch.Generator(device="cuda").manual_seed(1)
    pitch = 1504
    x = torch.randint(-127, 128, (600, pitch), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-127, 128, (n, pitch), generator=g, device="cuda", dtype=torch.int8)
    xs, ws = torch.rand(600, generator=g, device="cuda") / 500, torch.rand(n, generator=g, device="cuda")
    bias = torch.randn(n, generator=g, device="cuda")
    ys = []
    for rows in (1, 3, 8, 9, 64, 200, 256, 257, 600):
        y = torch.empty(rows, n, dtype=torch.float16, device="cuda")
        fx.i8_linear_dev(ptr(x), ptr(y), rows, n, k, ptr(w), ptr(ws), ptr(xs), "f16", x_stride=pitch, codes_stride=pitch,
                         bias_ptr=ptr(bias), stream=stream(torch))
        ys.append(y)
    torch.cuda.synchronize()
    for y in ys[:-1]:
        assert torch.equal(y, ys[-1][:y.shape[0]])


# ---- used together ----------------------------------------------------------------------------------------------


class Block:
    """Two projections with a layer norm before each: norm to int8 rows -> linear -> (residual) norm -> linear, weights
    quantised on the device from f32."""

    def __init__(self, torch, rows, k, n, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.torch, self.rows, self.k, self.n = torch, rows, k, n
        self.pitch, self.pitch2 = (k + 15) // 16 * 16, (n + 15) // 16 * 16
        self.w = torch.randn(n, k, generator=g, device="cuda") / k ** 0.5
        self.w2 = torch.randn(k, n, generator=g, device="cuda") / n ** 0.5
        self.x = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
        self.r = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
        self.gain = (torch.rand(k, generator=g, device="cuda") + 0.5).bfloat16()
        self.shift = torch.randn(k, generator=g, device="cuda").bfloat16()
        e = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
        self.codes, self.scales = e(n, self.pitch, dtype=torch.int8), e(n)
        self.codes2, self.scales2 = e(k, self.pitch2, dtype=torch.int8), e(k)
        self.sum, self.q, self.qs = torch.empty_like(self.x), e(rows, self.pitch, dtype=torch.int8), e(rows)
        self.y = e(rows, n, dtype=torch.bfloat16)
        self.q2, self.qs2 = e(rows, self.pitch2, dtype=torch.int8), e(rows)
        self.z = e(rows, k)

    def quantize(self):
        st = stream(self.torch)
        fx.i8_quantize_dev(ptr(self.w), self.n, self.k, ptr(self.codes), ptr(self.scales), "f32", codes_stride=self.pitch, stream=st)
        fx.i8_quantize_dev(ptr(self.w2), self.k, self.n, ptr(self.codes2), ptr(self.scales2), "f32", codes_stride=self.pitch2,
                           stream=st)

    def step(self):
        st = stream(self.torch)
        fx.layer_norm_dev(ptr(self.x), ptr(self.q), self.rows, self.k, "bf16", "i8", ptr(self.gain), ptr(self.shift),
                          residual_ptr=ptr(self.r), sum_ptr=ptr(self.sum), y_stride=self.pitch, scale_ptr=ptr(self.qs),
                          scale_mode="row", stream=st)
        fx.i8_linear_dev(ptr(self.q), ptr(self.y), self.rows, self.n, self.k, ptr(self.codes), ptr(self.scales), ptr(self.qs),
                         "bf16", x_stride=self.pitch, codes_stride=self.pitch, stream=st)
        fx.i8_quantize_dev(ptr(self.y), self.rows, self.n, ptr(self.q2), ptr(self.qs2), "bf16", codes_stride=self.pitch2, stream=st)
        fx.i8_linear_dev(ptr(self.q2), ptr(self.z), self.rows, self.k, self.n, ptr(self.codes2), ptr(self.scales2), ptr(self.qs2),
                         "f32", x_stride=self.pitch2, codes_stride=self.pitch2, stream=st)

    def check(self):
        from test_layer_norm_gpu import check_norm

        torch = self.torch
        for w, codes, scales in ((self.w, self.codes, self.scales), (self.w2, self.codes2, self.scales2)):
            want, sc = quantize_want(torch, w)
            assert torch.equal(codes[:, :w.shape[1]], want) and torch.equal(scales[:, None], sc)
        check_norm(torch, self.x, self.r, self.gain, self.shift, 1e-5, "i8", self.q[:, :self.k], self.qs, "row")
        assert torch.equal(self.y, linear_want(torch, self.q[:, :self.k], self.qs, self.codes[:, :self.k], self.scales, None, "bf16"))
        want, sc = quantize_want(torch, self.y)
        assert torch.equal(self.q2[:, :self.n], want) and torch.equal(self.qs2[:, None], sc)
        assert torch.equal(self.z, linear_want(torch, self.q2[:, :self.n], self.qs2, self.codes2[:, :self.n], self.scales2, None, "f32"))


@pytest.mark.parametrize("rows,k,n", [(1, 1024, 512), (4, 2048, 1000), (20, 510, 264), (200, 768, 3000), (700, 1000, 2048)])
def test_block_of_calls(cuda_torch, rows, k, n):
    b = Block(cuda_torch, rows, k, n)
    b.quantize()
    b.step()
    cuda_torch.cuda.synchronize()
    b.check()


@pytest.mark.parametrize("rows", [1, 6, 40, 200, 600])
def test_captured_replayed_and_side_by_side(cuda_torch, rows):
    """Two graphs of the same calls on two streams at once, replayed on new inputs, with eager calls between."""
    torch = cuda_torch
    blocks = [Block(torch, rows, 1024, 640, seed=s) for s in range(3)]
    streams = [torch.cuda.Stream() for _ in blocks]
    graphs = []
    torch.cuda.synchronize()
    for b, st in zip(blocks[:2], streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            b.quantize()
            b.step()
        graphs.append(g)
    for turn in range(3):
        for b in blocks:
            b.x.copy_(torch.randn_like(b.x.float()) * (turn + 1))
            b.w.copy_(torch.randn_like(b.w) * 0.1)
        torch.cuda.synchronize()
        for _ in range(4):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
            with torch.cuda.stream(streams[2]):
                blocks[2].quantize()
                blocks[2].step()
        torch.cuda.synchronize()
        for b in blocks:
            b.check()


def test_host_pointers_and_mixed_calls(cuda_torch):
    torch = cuda_torch
    d = torch.zeros(64, 64, device="cuda", dtype=torch.int8)
    f = torch.zeros(64, 64, device="cuda")
    h = torch.zeros(64, 64, dtype=torch.int8)
    for call in (lambda: fx.i8_linear_dev(ptr(h), ptr(f), 4, 8, 64, ptr(d), ptr(f), ptr(f), "f32"),
                 lambda: fx.i8_quantize_dev(ptr(f), 4, 64, ptr(h), ptr(f), "f32"),
                 lambda: fx.i8_dequantize_dev(ptr(h), ptr(f), 4, 64, ptr(f), "f32")):
        with pytest.raises(fx.FxError) as e:
            call()
        assert e.value.code == fx.FX_INVALID_ARGUMENT and "device memory" in str(e.value)
    run_linear(torch, 3, 64, 64)  # and the next call is served


def test_other_device(cuda_torch):
    torch = cuda_torch
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    with torch.cuda.device(1):
        x = torch.randint(-127, 128, (5, 256), device="cuda", dtype=torch.int8)
        w = torch.randint(-127, 128, (300, 256), device="cuda", dtype=torch.int8)
        xs, ws = torch.rand(5, device="cuda"), torch.rand(300, device="cuda")
        y = torch.empty(5, 300, device="cuda")
    with torch.cuda.device(0):
        fx.i8_linear_dev(ptr(x), ptr(y), 5, 300, 256, ptr(w), ptr(ws), ptr(xs), "f32")
        assert torch.cuda.current_device() == 0
    torch.cuda.synchronize(1)
    assert torch.equal(y, linear_want(torch, x, xs, w, ws, None, "f32"))


@pytest.mark.parametrize("rows", [3, 200, 700])
def test_captured_with_branches(cuda_torch, rows):
    """A graph whose calls follow calls of two streams, a copy and a fill: each sees what all of them wrote, eagerly and replayed."""
    torch = cuda_torch
    k, n = 1024, 1536
    g = torch.Generator(device="cuda").manual_seed(rows)
    h = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
    w = torch.randn(n, k, generator=g, device="cuda")
    q, qs = torch.zeros(rows, k, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    codes, scales = torch.zeros(n, k, dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda")
    y, z, back = torch.zeros(rows, n, device="cuda"), torch.zeros(rows, n, device="cuda"), torch.zeros(n, k, device="cuda")
    side = torch.cuda.Stream()

    def step():
        here = torch.cuda.current_stream()
        q.zero_()
        codes.zero_()
        side.wait_stream(here)
        fx.layer_norm_dev(ptr(h), ptr(q), rows, k, "bf16", "i8", scale_ptr=ptr(qs), scale_mode="row", stream=stream(torch))
        with torch.cuda.stream(side):
            fx.i8_quantize_dev(ptr(w), n, k, ptr(codes), ptr(scales), "f32", stream=stream(torch))
        here.wait_stream(side)
        fx.i8_linear_dev(ptr(q), ptr(y), rows, n, k, ptr(codes), ptr(scales), ptr(qs), "f32", stream=stream(torch))
        side.wait_stream(here)
        with torch.cuda.stream(side):
            fx.i8_dequantize_dev(ptr(codes), ptr(scales), n, k, ptr(back), "f32", stream=stream(torch))
        z.copy_(y)
        y.fill_(-1.0)
        fx.i8_linear_dev(ptr(q), ptr(y), rows, n, k, ptr(codes), ptr(scales), ptr(qs), "f32", stream=stream(torch))
        here.wait_stream(side)

    def check():
        torch.cuda.synchronize()
        want_codes, sc = quantize_want(torch, w)
        assert torch.equal(codes, want_codes) and torch.equal(back, want_codes.float() * sc)
        want = linear_want(torch, q, qs, codes, scales, None, "f32")
        assert bool(q.any()) and torch.equal(y, want) and torch.equal(z, want)

    for _ in range(3):
        step()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        h.copy_(torch.randn(rows, k, generator=g, device="cuda") * (i + 1))
        w.copy_(torch.randn(n, k, generator=g, device="cuda"))
        for _ in range(4):
            graph.replay()
        check()
