"""Measured cases of the 8-bit integer linear layer with its quantiser, and of the layer norm with its backward pass.

`run` computes a case either in its plain form (elementary torch operations in 32 bits, rounded once at the end) or,
with `own` set, by the library's entry points. `exact` computes it from the definitions in 64 bits."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "i8": 1}
TOP = {"e4m3": 448.0, "i8": 127.0}  # the largest value of an 8-bit type
AMAX_FLOOR = 1e-30  # the largest magnitude of a row counts as at least this when its scale is made
EPS = 1e-5


def _norm(name, rows, cols, x, y, residual=True, scale="row", stats=False):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "x": x, "y": y, "residual": residual,
            "scale": scale if y in TOP else "", "stats": stats}


def _backward(name, rows, cols, t, dsum=True):
    return {"name": name, "op": "backward", "rows": rows, "cols": cols, "type": t, "dsum": dsum}


def _linear(name, rows, k, n, y, bias=False, scale="row", pad=16):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "y": y, "bias": bias, "scale": scale, "pad": pad}


def _quantize(name, rows, cols, x):
    return {"name": name, "op": "quantize", "rows": rows, "cols": cols, "x": x}


def _chain(name, rows, k, n):
    return {"name": name, "op": "chain", "rows": rows, "k": k, "n": n}


def listed():
    return [
        # one token's norm before an 8-bit projection: launch latency
        _norm("norm, one token", 1, 4096, "bf16", "e4m3"),
        # a whole prompt (or the patch tokens of a batch of tiles) on its way through a model that is trained
        _norm("norm, 16384 tokens", 16384, 4096, "bf16", "bf16", stats=True),
        # the same training step's way back, with the gradient that arrives beside the norm
        _backward("backward, 8192 tokens", 8192, 4096, "bf16"),
        # rows that are no multiple of a vector
        _backward("backward, odd rows", 1031, 5119, "f16", dsum=False),
        # a single token through an attention projection
        _linear("linear, one token", 1, 4096, 4096, "bf16"),
        # a few sequences decoded together through a wide up-projection: the weights come from memory
        _linear("linear, 8 tokens, wide", 8, 8192, 28672, "f16"),
        # a large decoding batch
        _linear("linear, 192 tokens", 192, 8192, 8192, "bf16", bias=True),
        # a ragged prompt against odd extents, rows of codes laid out 16 bytes apart
        _linear("linear, 1003 tokens, odd", 1003, 4705, 5003, "f16", bias=True),
        # a prompt through an up-projection: the tensor cores' rate
        _linear("linear, 4096 tokens", 4096, 4096, 14336, "bf16"),
        # a stored f32 layer made 8-bit and read back, as at loading
        _quantize("quantise, f32", 8192, 8192, "f32"),
        # a batch of 16-bit activations
        _quantize("quantise, small", 1003, 1088, "bf16"),
        # one decoding step of a block: residual, norm, 8-bit projection
        _chain("norm and linear, 4 tokens", 4, 4096, 11008),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "backward", "backward", "linear", "linear", "linear", "quantize", "chain"])
    if op in ("norm", "backward", "quantize"):
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.6:
            cols = max(64, cols // 64 * 64)
        rows = max(1, min(_log(rng, 1, 200000), (60_000_000 if op != "backward" else 30_000_000) // cols))
        t = rng.choice(["bf16", "f16", "f32"])
        if op == "norm":
            y = rng.choice(["e4m3", "i8", "bf16", "f16", "f32"])
            c = _norm("", rows, cols, t, y, rng.random() < 0.7, rng.choice(["row", "row", "tensor"]), rng.random() < 0.4)
        elif op == "backward":
            c = _backward("", rows, cols, t, rng.random() < 0.5)
        else:
            c = _quantize("", rows, cols, t)
    else:
        k = _log(rng, 256, 16384)
        if rng.random() < 0.6:
            k = k // 64 * 64
        n = min(_log(rng, 64, 28672), 230_000_000 // k)
        if rng.random() < 0.5:
            n = max(64, n // 64 * 64)
        rows = min(_log(rng, 1, 4096) if rng.random() < 0.6 else rng.randint(1, 16), 200_000_000_000 // (n * k))
        if op == "linear":
            c = _linear("", max(1, rows), k, n, rng.choice(["bf16", "f16", "f32"]), rng.random() < 0.5,
                        rng.choice(["row", "row", "tensor"]), 1 if rng.random() < 0.1 else 16)
        else:
            c = _chain("", max(1, min(rows, 64)), k, n)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------


def _tokens(g, rows, cols):
    """Activations: unit-variance values around a mean of their row, one channel in 64 sixteen times as large, as hidden
    states have them."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    loud = torch.rand(cols, generator=g, device="cuda") < 1 / 64
    return x * torch.where(loud, 16.0, 1.0) + 0.5 * torch.randn(rows, 1, generator=g, device="cuda")


def _weights(g, n, k):
    return torch.randn(n, k, generator=g, device="cuda") * (torch.rand(n, 1, generator=g, device="cuda") + 0.5) / math.sqrt(k)


def _pitch(k, pad):
    return (k + pad - 1) // pad * pad


def _codes(v, pad):
    """(codes [rows][cols] in rows a multiple of `pad` apart, scales [rows]) of f32 rows."""
    scale = v.abs().amax(1).clamp(min=AMAX_FLOOR) / TOP["i8"]
    q = torch.zeros(v.shape[0], _pitch(v.shape[1], pad), dtype=torch.int8, device="cuda")[:, :v.shape[1]]
    q.copy_(torch.round(v / scale[:, None]).clamp(-TOP["i8"], TOP["i8"]))
    return q, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    op = case["op"]
    if op in ("norm", "chain"):
        rows, cols = case["rows"], case["cols"] if op == "norm" else case["k"]
        t = TYPES[case.get("x", "bf16")]
        s["x"] = _tokens(g, rows, cols).to(t)
        s["weight"] = (1.0 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(t)
        s["bias"] = (0.1 * torch.randn(cols, generator=g, device="cuda")).to(t)
        if op == "chain" or case["residual"]:
            s["residual"] = (3.0 * _tokens(g, rows, cols)).to(t)
        if case.get("scale") == "tensor":
            s["scale"] = torch.full((1,), (4.0 + seed % 7) / TOP[case["y"]], device="cuda")
    if op == "backward":
        rows, cols, t = case["rows"], case["cols"], TYPES[case["type"]]
        h = (3.0 * _tokens(g, rows, cols)).to(t)
        s["h"] = h
        f = h.float()
        s["mean"] = f.mean(1)
        s["rstd"] = 1.0 / torch.sqrt((f - s["mean"][:, None]).square().mean(1) + EPS)
        s["weight"] = (1.0 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(t)
        s["dy"] = torch.randn(rows, cols, generator=g, device="cuda").to(t)
        if case["dsum"]:
            s["dsum"] = torch.randn(rows, cols, generator=g, device="cuda").to(t)
    if op == "linear":
        x, scale = _codes(_tokens(g, case["rows"], case["k"]), case["pad"])
        s["x"], s["x_scale"] = x, scale if case["scale"] == "row" else scale.mean().reshape(1)
    if op in ("linear", "chain"):
        s["codes"], s["scales"] = _codes(_weights(g, case["n"], case["k"]), case.get("pad", 16))
        if case.get("bias"):
            s["y_bias"] = torch.randn(case["n"], generator=g, device="cuda")
    if op == "quantize":
        s["w"] = _weights(g, case["rows"], case["cols"]).to(TYPES[case["x"]])
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------


def _plain_norm(s, y_type, stats):
    """Outputs of the norm; an 8-bit y as f32 whole numbers or e4m3 values in f32, before its scale."""
    x, scale = s["x"], s.get("scale")
    h = x.float()
    out = {}
    if "residual" in s:
        h = h + s["residual"].float()
        out["sum"] = h.to(x.dtype)
    mean = h.mean(1, keepdim=True)
    c = h - mean
    rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    if stats:
        out["mean"], out["rstd"] = mean[:, 0], rstd[:, 0]
    y = c * rstd * s["weight"].float() + s["bias"].float()
    if y_type in TOP:
        if scale is None:
            scale = y.abs().amax(1).clamp(min=AMAX_FLOOR) / TOP[y_type]
            out["scale"] = scale
            scale = scale[:, None]
        y = (y / scale).clamp(-TOP[y_type], TOP[y_type])
    out["y"] = torch.round(y) if y_type == "i8" else y.to(TYPES[y_type])
    return out


def _plain_linear(s, x, x_scale, y_type):
    y = x.float() @ s["codes"].float().t()
    y = y * x_scale[:, None] * s["scales"]
    if "y_bias" in s:
        y = y + s["y_bias"]
    return y.to(TYPES[y_type])


def _plain(s):
    case = s["case"]
    if case["op"] == "norm":
        out = _plain_norm(s, case["y"], case["stats"])
        if case["y"] == "i8":  # as the values it stands for
            out["y"] = (out["y"] * out.get("scale", s.get("scale"))[:, None]).to(torch.bfloat16)
        return out
    if case["op"] == "backward":
        xhat = (s["h"].float() - s["mean"][:, None]) * s["rstd"][:, None]
        dy = s["dy"].float()
        g = dy * s["weight"].float()
        dx = (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True)) * s["rstd"][:, None]
        if "dsum" in s:
            dx = dx + s["dsum"].float()
        return {"dx": dx.to(s["h"].dtype), "dweight": (dy * xhat).sum(0), "dbias": dy.sum(0)}
    if case["op"] == "linear":
        return {"y": _plain_linear(s, s["x"], s["x_scale"], case["y"])}
    if case["op"] == "chain":
        h = _plain_norm(s, "i8", False)
        return {"sum": h["sum"], "y": _plain_linear(s, h["y"], h["scale"], "bf16")}
    w = s["w"].float()
    scale = w.abs().amax(1).clamp(min=AMAX_FLOOR) / TOP["i8"]
    q = torch.round(w / scale[:, None]).clamp(-TOP["i8"], TOP["i8"])
    return {"scale": scale, "values": (q * scale[:, None]).to(torch.bfloat16)}


# ---- the library's calls ---------------------------------------------------------------------------------------


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_norm(s, y_type, stats):
    import fenix_b200 as fx

    x, residual, scale = s["x"], s.get("residual"), s.get("scale")
    rows, cols = x.shape
    t = s["case"].get("x", "bf16")
    mode = None if y_type not in TOP else "tensor" if scale is not None else "row"
    pitch = _pitch(cols, 16) if y_type == "i8" else cols
    out = {"y": torch.empty(rows, pitch, dtype=torch.int8 if y_type == "i8" else TYPES[y_type], device="cuda")}
    if mode == "row":
        out["scale"] = scale = torch.empty(rows, device="cuda")
    if residual is not None:
        out["sum"] = torch.empty_like(x)
    if stats:
        out["mean"], out["rstd"] = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    fx.layer_norm_dev(x.data_ptr(), out["y"].data_ptr(), rows, cols, x_type=t, y_type=y_type,
                      weight_ptr=s["weight"].data_ptr(), bias_ptr=s["bias"].data_ptr(), weight_type=t, eps=EPS,
                      residual_ptr=_ptr(residual), residual_type=t, sum_ptr=_ptr(out.get("sum")), y_stride=pitch,
                      mean_ptr=_ptr(out.get("mean")), rstd_ptr=_ptr(out.get("rstd")), scale_ptr=_ptr(scale),
                      scale_mode=mode, stream=_stream())
    return out


def _own_linear(s, x, x_scale, x_stride, y_type, mode):
    import fenix_b200 as fx

    case = s["case"]
    rows, n = case["rows"], case["n"]
    y = torch.empty(rows, n, dtype=TYPES[y_type], device="cuda")
    fx.i8_linear_dev(x.data_ptr(), y.data_ptr(), rows, n, case["k"], s["codes"].data_ptr(), s["scales"].data_ptr(),
                     x_scale.data_ptr(), y_type=y_type, x_scale_mode=mode, x_stride=x_stride,
                     codes_stride=s["codes"].stride(0), bias_ptr=_ptr(s.get("y_bias")), stream=_stream())
    return y


def _own_values(codes, scale, mode, rows, cols, stride):
    import fenix_b200 as fx

    values = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    fx.i8_dequantize_dev(codes.data_ptr(), scale.data_ptr(), rows, cols, values.data_ptr(), y_type="bf16",
                         scale_mode=mode, codes_stride=stride, stream=_stream())
    return values


def _own(s):
    import fenix_b200 as fx

    case = s["case"]
    if case["op"] == "norm":
        out = _own_norm(s, case["y"], case["stats"])
        if case["y"] == "i8":
            out["y"] = _own_values(out["y"], out.get("scale", s.get("scale")), case["scale"], case["rows"], case["cols"],
                                   out["y"].stride(0))
        return out
    if case["op"] == "backward":
        h, t = s["h"], case["type"]
        rows, cols = h.shape
        dx = torch.empty_like(h)
        dweight, dbias = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
        work = torch.empty(fx.layer_norm_backward_workspace(rows, cols), dtype=torch.uint8, device="cuda")
        fx.layer_norm_backward_dev(s["dy"].data_ptr(), h.data_ptr(), s["mean"].data_ptr(), s["rstd"].data_ptr(), rows,
                                   cols, dy_type=t, h_type=t, weight_ptr=s["weight"].data_ptr(), weight_type=t,
                                   dsum_ptr=_ptr(s.get("dsum")), dx_ptr=dx.data_ptr(), dx_type=t,
                                   dweight_ptr=dweight.data_ptr(), dbias_ptr=dbias.data_ptr(), work_ptr=work.data_ptr(),
                                   work_bytes=work.numel(), stream=_stream())
        return {"dx": dx, "dweight": dweight, "dbias": dbias}
    if case["op"] == "linear":
        return {"y": _own_linear(s, s["x"], s["x_scale"], s["x"].stride(0), case["y"], case["scale"])}
    if case["op"] == "chain":
        h = _own_norm(s, "i8", False)
        return {"sum": h["sum"], "y": _own_linear(s, h["y"], h["scale"], h["y"].stride(0), "bf16", "row")}
    rows, cols = case["rows"], case["cols"]
    pitch = _pitch(cols, 16)
    codes = torch.empty(rows, pitch, dtype=torch.int8, device="cuda")
    scale = torch.empty(rows, device="cuda")
    fx.i8_quantize_dev(s["w"].data_ptr(), rows, cols, codes.data_ptr(), scale.data_ptr(), x_type=case["x"],
                       scale_mode="row", codes_stride=pitch, stream=_stream())
    return {"scale": scale, "values": _own_values(codes, scale, "row", rows, cols, pitch)}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---- work and the definitions in 64 bits -----------------------------------------------------------------------


def _norm_bytes(rows, cols, x, y, residual, stats):
    per = SIZE[x] * (3 if residual else 1) + SIZE[y]
    return rows * cols * per + 2 * cols * SIZE[x] + (4 * rows if y in TOP else 0) + (8 * rows if stats else 0)


def work(case):
    op, rows = case["op"], case["rows"]
    if op == "norm":
        back = rows * case["cols"] * 3 if case["y"] == "i8" else 0  # its values read back
        return {"bytes": _norm_bytes(rows, case["cols"], case["x"], case["y"], case["residual"], case["stats"]) + back,
                "flops": 9 * rows * case["cols"]}
    if op == "backward":
        cols, size = case["cols"], SIZE[case["type"]]
        return {"bytes": rows * cols * size * (4 if case["dsum"] else 3) + cols * (size + 8) + 8 * rows,
                "flops": 14 * rows * cols}
    if op == "quantize":
        return {"bytes": rows * case["cols"] * (SIZE[case["x"]] + 4) + 8 * rows, "flops": 4 * rows * case["cols"]}
    n, k = case["n"], case["k"]
    flops = 2 * rows * n * k
    if op == "chain":
        return {"bytes": rows * k * 6 + 4 * k + n * k + 4 * n + rows * n * 2, "flops": flops + 9 * rows * k}
    extra = 4 * n * (2 if case["bias"] else 1) + (4 * rows if case["scale"] == "row" else 4)
    return {"bytes": rows * k + n * k + rows * n * SIZE[case["y"]] + extra, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    d = torch.float64

    def norm(y_type):
        h = s["x"].to(d)
        r = {}
        if "residual" in s:
            h = h + s["residual"].to(d)
            r["sum"] = h
        var, mean = torch.var_mean(h, dim=1, correction=0, keepdim=True)
        inv = torch.rsqrt(var + EPS)
        if case.get("stats"):
            r["mean"], r["rstd"] = mean.flatten(), inv.flatten()
        y = torch.addcmul(s["bias"].to(d), (h - mean) * inv, s["weight"].to(d))
        if y_type in TOP:
            if "scale" in s:
                scale = s["scale"].to(d)
            else:
                scale = torch.linalg.vector_norm(y, ord=float("inf"), dim=1, keepdim=True).clamp(min=AMAX_FLOOR) / TOP[y_type]
                r["scale"] = scale.flatten()
            y = torch.clamp(y / scale, -TOP[y_type], TOP[y_type])
            if y_type == "i8":  # the rounding to whole numbers belongs to the definition
                r["codes"], y = torch.round(y), torch.round(y) * scale
        r["y"] = y  # before its rounding to a floating type
        return r

    if op == "norm":
        r = norm(case["y"])
        r.pop("codes", None)
        return r
    if op == "backward":
        h, dy, inv = s["h"].to(d), s["dy"].to(d), s["rstd"].to(d)[:, None]
        z = torch.sub(h, s["mean"].to(d)[:, None]) * inv
        v = dy * s["weight"].to(d)
        n = h.shape[1]
        dx = torch.addcmul(v - v.sum(1, keepdim=True) / n, z, torch.einsum("rc,rc->r", v, z)[:, None] / n, value=-1) * inv
        if "dsum" in s:
            dx = dx + s["dsum"].to(d)
        return {"dx": dx, "dweight": torch.einsum("rc,rc->c", dy, z), "dbias": torch.einsum("rc->c", dy)}
    if op == "quantize":
        w = s["w"].to(d)
        sc = torch.linalg.vector_norm(w, ord=float("inf"), dim=1, keepdim=True).clamp(min=AMAX_FLOOR) / TOP["i8"]
        return {"scale": sc.flatten(), "values": torch.round(w / sc.float().to(d)).clamp(-127, 127) * sc}
    w = s["codes"].to(d) * s["scales"].to(d)[:, None]
    if op == "chain":
        h = norm("i8")
        return {"sum": h["sum"], "y": torch.matmul(h["codes"] * h["scale"][:, None], w.T)}
    y = torch.matmul(s["x"].to(d), w.T) * s["x_scale"].to(d)[:, None]
    return {"y": y + s["y_bias"].to(d) if "y_bias" in s else y}
