"""The token operators' measured cases: the root-mean-square norm with the residual's addition and 8-bit output,
the linear layer with 4-bit weights and group scales, and the quantiser that makes such weights.

`run` computes a case either in its plain form (elementary torch operations in 32 bits, rounded once at the end) or,
with `own` set, by the library's entry points. `exact` computes it from the definitions in 64 bits."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
E4M3_MAX = 448.0
AMAX_FLOOR = 1e-30  # the largest magnitude of a row counts as at least this when its scale is made
EPS = 1e-5
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}


def _norm(name, rows, cols, x, y, residual=True, scale="row"):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "x": x, "y": y, "residual": residual,
            "scale": scale if y == "e4m3" else ""}


def _linear(name, rows, k, n, group, x, y, zeros=False, bias=False):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "group": group, "x": x, "y": y, "zeros": zeros,
            "bias": bias}


def _quantize(name, n, k, group, w, zeros=False):
    return {"name": name, "op": "quantize", "n": n, "k": k, "group": group, "w": w, "zeros": zeros}


def _chain(name, rows, k, n, group, zeros=False):
    return {"name": name, "op": "chain", "rows": rows, "k": k, "n": n, "group": group, "zeros": zeros}


def listed():
    return [
        # one token's norm before a projection: launch latency
        _norm("norm, one token", 1, 4096, "bf16", "e4m3"),
        # a whole prompt (or the patch tokens of a batch of tiles) normalised for 8-bit products
        _norm("norm, 16384 tokens", 16384, 4096, "bf16", "e4m3"),
        # rows that are no multiple of a vector, a calibrated scale for the whole tensor
        _norm("norm, odd rows", 1031, 5119, "f16", "e4m3", scale="tensor"),
        # a single token through an attention projection
        _linear("linear, one token", 1, 4096, 4096, 128, "bf16", "bf16"),
        # a single token through a wide up-projection: the weights come from memory
        _linear("linear, one token, wide", 1, 8192, 28672, 128, "f16", "f16"),
        # a few sequences decoded together, 8-bit activations, zero points, small groups
        _linear("linear, 8 tokens", 8, 4096, 14336, 64, "e4m3", "bf16", zeros=True),
        # a ragged batch against odd extents
        _linear("linear, 37 tokens, odd", 37, 4704, 5003, 32, "bf16", "bf16", zeros=True, bias=True),
        # a large decoding batch
        _linear("linear, 192 tokens", 192, 8192, 8192, 128, "f16", "f16", bias=True),
        # a prompt through an up-projection: the tensor cores' rate
        _linear("linear, 4096 tokens", 4096, 4096, 14336, 128, "bf16", "bf16"),
        # a stored f32 layer made 4-bit and read back, as at loading
        _quantize("quantise, f32", 8192, 8192, 128, "f32"),
        # a narrow 16-bit layer with zero points
        _quantize("quantise, small, zeros", 1003, 1088, 32, "bf16", zeros=True),
        # one decoding step of a block: residual, norm, 8-bit projection
        _chain("norm and linear, 4 tokens", 4, 4096, 11008, 128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "linear", "linear", "linear", "quantize", "chain"])
    if op == "norm":
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.6:
            cols = max(64, cols // 64 * 64)
        rows = min(_log(rng, 1, 200000), 60_000_000 // cols)
        y = rng.choice(["e4m3", "e4m3", "bf16", "f16", "f32"])
        c = _norm("", max(1, rows), cols, rng.choice(["bf16", "f16", "f32"]), y, rng.random() < 0.7,
                  rng.choice(["row", "row", "tensor"]))
    elif op == "quantize":
        group = rng.choice([32, 64, 128, 256])
        k = max(1, _log(rng, 256, 16384) // group) * group
        n = min(_log(rng, 32, 16384), 60_000_000 // k)
        c = _quantize("", max(1, n), k, group, rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.5)
    else:
        group = rng.choice([32, 64, 128, 128, 256])
        k = max(1, _log(rng, 512, 16384) // group) * group
        n = min(_log(rng, 64, 28672), 200_000_000 // k)
        if rng.random() < 0.5:
            n = max(64, n // 64 * 64)
        rows = min(_log(rng, 1, 4096) if rng.random() < 0.6 else rng.randint(1, 16), 200_000_000_000 // (n * k))
        if op == "linear":
            c = _linear("", max(1, rows), k, n, group, rng.choice(["bf16", "f16", "e4m3"]),
                        rng.choice(["bf16", "f16"]), rng.random() < 0.5, rng.random() < 0.5)
        else:
            c = _chain("", max(1, min(rows, 64)), k, n, group, rng.random() < 0.5)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------


def _tokens(g, rows, cols):
    """Activations: unit-variance values with one channel in 64 sixteen times as large, as hidden states have them."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    loud = torch.rand(cols, generator=g, device="cuda") < 1 / 64
    return x * torch.where(loud, 16.0, 1.0)


def _weights(g, n, k):
    return torch.randn(n, k, generator=g, device="cuda") * (torch.rand(n, 1, generator=g, device="cuda") + 0.5) / math.sqrt(k)


def _groups(w, group, zeros):
    """(integer codes 0..15, scales f16, zero points or None) of f32 weights [n][k]: the values w takes are
    scale * (code - zero), zero = 8 without zero points."""
    n, k = w.shape
    v = w.view(n, k // group, group)
    if zeros:
        lo, hi = v.amin(2).clamp(max=0.0), v.amax(2).clamp(min=0.0)
        s = ((hi - lo) / torch.full_like(hi, 15.0)).half()
        d = s.float()
        z = torch.where(d > 0, torch.round(-lo / d), torch.zeros_like(lo)).clamp(0, 15)
    else:
        s = (v.abs().amax(2) / torch.full((), 7.0, device=w.device)).half()
        d = s.float()
        z = torch.full_like(d, 8.0)
    q = torch.where(d[..., None] > 0, torch.round(v / d[..., None]), torch.zeros_like(v))
    q = (q + z[..., None]).clamp(0, 15)
    return q.to(torch.uint8).view(n, k), s, z.to(torch.uint8) if zeros else None


def _packed(g, case):
    codes, scales, zeros = _groups(_weights(g, case["n"], case["k"]), case["group"], case["zeros"])
    return codes[:, 0::2] | (codes[:, 1::2] << 4), scales, zeros


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    op = case["op"]
    if op in ("norm", "chain"):
        rows, cols = case["rows"], case["cols"] if op == "norm" else case["k"]
        t = TYPES[case.get("x", "bf16")]
        s["x"] = _tokens(g, rows, cols).to(t)
        s["weight"] = (1.0 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(t)
        if op == "chain" or case["residual"]:
            s["residual"] = (3.0 * _tokens(g, rows, cols)).to(t)
        if case.get("scale") == "tensor":
            s["scale"] = torch.full((1,), 0.01 + 0.02 * (seed % 7) / 7, device="cuda")
    if op == "linear":
        x = _tokens(g, case["rows"], case["k"])
        if case["x"] == "e4m3":
            amax = x.abs().amax(1)
            s["x_scale"] = amax / E4M3_MAX
            x = (x * (E4M3_MAX / amax)[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        s["x"] = x.to(TYPES[case["x"]])
        if case["bias"]:
            s["bias"] = torch.randn(case["n"], generator=g, device="cuda")
    if op in ("linear", "chain"):
        s["codes"], s["scales"], s["zeros"] = _packed(g, case)
    if op == "quantize":
        s["w"] = _weights(g, case["n"], case["k"]).to(TYPES[case["w"]])
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------


def _plain_norm(x, residual, weight, y_type, scale):
    h = x.float()
    out = {}
    if residual is not None:
        h = h + residual.float()
        out["sum"] = h.to(x.dtype)
    y = h * (1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)) * weight.float()
    if y_type == "e4m3":
        if scale is None:
            scale = y.abs().amax(1).clamp(min=AMAX_FLOOR) / E4M3_MAX
            out["scale"] = scale
            scale = scale[:, None]
        y = (y / scale).clamp(-E4M3_MAX, E4M3_MAX)
    out["y"] = y.to(TYPES[y_type])
    return out


def _values(codes, scales, zeros, group, t):
    """The weights [n][k] that packed codes stand for, in torch type t."""
    n, k = codes.shape[0], 2 * codes.shape[1]
    c = torch.stack((codes & 15, codes >> 4), 2).view(n, k // group, group).to(t)
    z = zeros.to(t)[..., None] if zeros is not None else 8.0
    return ((c - z) * scales.to(t)[..., None]).view(n, k)


def _plain_linear(s, x, x_scale, y_type):
    case = s["case"]
    y = x.float() @ _values(s["codes"], s["scales"], s["zeros"], case["group"], torch.float32).t()
    if x_scale is not None:
        y = y * x_scale[:, None]
    if s.get("bias") is not None:
        y = y + s["bias"]
    return y.to(TYPES[y_type])


def _plain(s):
    case = s["case"]
    if case["op"] == "norm":
        return _plain_norm(s["x"], s.get("residual"), s["weight"], case["y"], s.get("scale"))
    if case["op"] == "linear":
        return {"y": _plain_linear(s, s["x"], s.get("x_scale"), case["y"])}
    if case["op"] == "chain":
        h = _plain_norm(s["x"], s["residual"], s["weight"], "e4m3", None)
        return {"sum": h["sum"], "y": _plain_linear(s, h["y"], h["scale"], "bf16")}
    codes, scales, zeros = _groups(s["w"].float(), case["group"], case["zeros"])
    z = zeros.float()[..., None] if zeros is not None else 8.0
    v = (codes.view(*scales.shape, case["group"]).float() - z) * scales.float()[..., None]
    return {"scales": scales, "values": v.view(s["w"].shape).to(s["w"].dtype)}


# ---- the library's calls ---------------------------------------------------------------------------------------


def _own_norm(s, x, y_type):
    import fenix_b200 as fx

    case, residual, scale = s["case"], s.get("residual"), s.get("scale")
    rows, cols = x.shape
    t = case.get("x", "bf16")
    out = {"y": torch.empty(rows, cols, dtype=TYPES[y_type], device="cuda")}
    mode = None
    if y_type == "e4m3":
        mode = "tensor" if scale is not None else "row"
        if scale is None:
            out["scale"] = scale = torch.empty(rows, device="cuda")
    if residual is not None:
        out["sum"] = torch.empty_like(x)
    fx.rms_norm_dev(x.data_ptr(), out["y"].data_ptr(), rows, cols, x_type=t, y_type=y_type,
                    weight_ptr=s["weight"].data_ptr(), weight_type=t, eps=EPS,
                    residual_ptr=residual.data_ptr() if residual is not None else None, residual_type=t,
                    sum_ptr=out["sum"].data_ptr() if residual is not None else None,
                    scale_ptr=scale.data_ptr() if mode else None, scale_mode=mode,
                    stream=torch.cuda.current_stream().cuda_stream)
    return out


def _own_linear(s, x, x_type, x_scale, y_type):
    import fenix_b200 as fx

    case, zeros, bias = s["case"], s["zeros"], s.get("bias")
    rows = x.shape[0]
    y = torch.empty(rows, case["n"], dtype=TYPES[y_type], device="cuda")
    fx.w4_linear_dev(x.data_ptr(), y.data_ptr(), rows, case["n"], case["k"], case["group"], s["codes"].data_ptr(),
                     s["scales"].data_ptr(), zeros_ptr=zeros.data_ptr() if zeros is not None else None,
                     x_type=x_type, y_type=y_type, scale_type="f16",
                     x_scale_ptr=x_scale.data_ptr() if x_scale is not None else None,
                     x_scale_mode="row" if x_scale is not None else None,
                     bias_ptr=bias.data_ptr() if bias is not None else None,
                     stream=torch.cuda.current_stream().cuda_stream)
    return y


def _own(s):
    import fenix_b200 as fx

    case = s["case"]
    if case["op"] == "norm":
        return _own_norm(s, s["x"], case["y"])
    if case["op"] == "linear":
        return {"y": _own_linear(s, s["x"], case["x"], s.get("x_scale"), case["y"])}
    if case["op"] == "chain":
        h = _own_norm(s, s["x"], "e4m3")
        return {"sum": h["sum"], "y": _own_linear(s, h["y"], "e4m3", h["scale"], "bf16")}
    n, k, group = case["n"], case["k"], case["group"]
    codes = torch.empty(n, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(n, k // group, dtype=torch.float16, device="cuda")
    zeros = torch.empty(n, k // group, dtype=torch.uint8, device="cuda") if case["zeros"] else None
    values = torch.empty_like(s["w"])
    zp, st = zeros.data_ptr() if zeros is not None else None, torch.cuda.current_stream().cuda_stream
    fx.w4_quantize_dev(s["w"].data_ptr(), n, k, group, codes.data_ptr(), scales.data_ptr(), zeros_ptr=zp,
                       w_type=case["w"], scale_type="f16", stream=st)
    fx.w4_dequantize_dev(codes.data_ptr(), scales.data_ptr(), n, k, group, values.data_ptr(), zeros_ptr=zp,
                         w_type=case["w"], scale_type="f16", stream=st)
    return {"scales": scales, "values": values}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---- work and the definitions in 64 bits -----------------------------------------------------------------------


def _norm_bytes(rows, cols, x, y, residual):
    per = SIZE[x] * (3 if residual else 1) + SIZE[y]
    return rows * cols * per + cols * SIZE[x] + (4 * rows if y == "e4m3" else 0)


def _code_bytes(case):
    groups = case["n"] * case["k"] // case["group"]
    return case["n"] * case["k"] // 2 + groups * (3 if case["zeros"] else 2)


def work(case):
    op = case["op"]
    if op == "norm":
        return {"bytes": _norm_bytes(case["rows"], case["cols"], case["x"], case["y"], case["residual"]),
                "flops": 6 * case["rows"] * case["cols"]}
    if op == "quantize":
        return {"bytes": 2 * (_code_bytes(case) + case["n"] * case["k"] * SIZE[case["w"]]),
                "flops": 6 * case["n"] * case["k"]}
    rows, n, k = case["rows"], case["n"], case["k"]
    flops = 2 * rows * n * k
    if op == "chain":
        return {"bytes": rows * k * 6 + 2 * k + _code_bytes(case) + rows * n * 2, "flops": flops + 6 * rows * k}
    extra = (4 * rows if case["x"] == "e4m3" else 0) + (4 * n if case["bias"] else 0)
    return {"bytes": rows * k * SIZE[case["x"]] + _code_bytes(case) + rows * n * 2 + extra, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    d = torch.float64

    def norm(quant):
        h = s["x"].to(d)
        r = {}
        if "residual" in s:
            h = h + s["residual"].to(d)
            r["sum"] = h
        ms = torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / h.shape[1]
        y = h * s["weight"].to(d) / torch.sqrt(ms + EPS)
        if quant == "row":
            r["scale"] = torch.clamp(torch.linalg.vector_norm(y, ord=float("inf"), dim=1), min=AMAX_FLOOR) / E4M3_MAX
            y = y / r["scale"][:, None]
        elif quant == "tensor":
            y = torch.clamp(y / s["scale"].to(d), -E4M3_MAX, E4M3_MAX)
        r["y"] = y  # before its rounding to 8 or 16 bits
        return r

    def weights():
        n, k, group = case["n"], case["k"], case["group"]
        w = torch.empty(n, k, dtype=d, device="cuda")
        w[:, 0::2] = (s["codes"] % 16).to(d)
        w[:, 1::2] = torch.div(s["codes"], 16, rounding_mode="floor").to(d)
        zero = s["zeros"].to(d) if s["zeros"] is not None else torch.full(s["scales"].shape, 8.0, dtype=d, device="cuda")
        w -= zero.repeat_interleave(group, dim=1)
        w *= s["scales"].to(d).repeat_interleave(group, dim=1)
        return w

    if op == "norm":
        return norm(case["scale"])
    if op == "linear":
        x = s["x"].to(torch.float32).to(d)
        if "x_scale" in s:
            x = x * s["x_scale"].to(d)[:, None]
        y = torch.matmul(x, weights().T)
        return {"y": y + s["bias"].to(d) if "bias" in s else y}
    if op == "chain":
        h = norm("row")
        # the product's operand is the norm's 8-bit output, so its rounding belongs to the definition
        q = h["y"].to(torch.float32).to(torch.float8_e4m3fn).to(torch.float32).to(d) * h["scale"][:, None]
        return {"sum": h["sum"], "y": torch.matmul(q, weights().T)}
    w = s["w"].to(d)
    n, k = w.shape
    v = w.reshape(-1, case["group"])
    if case["zeros"]:
        lo, hi = torch.clamp(v.min(1).values, max=0), torch.clamp(v.max(1).values, min=0)
        sc = ((hi - lo) / 15).to(torch.float16).to(d)[:, None]
        z = torch.where(sc > 0, torch.clamp(torch.round(-lo[:, None] / sc), 0, 15), torch.zeros_like(sc))
    else:
        sc = (torch.linalg.vector_norm(v, ord=float("inf"), dim=1) / 7).to(torch.float16).to(d)[:, None]
        z = torch.full_like(sc, 8)
    q = torch.where(sc > 0, torch.clamp(torch.round(v / sc) + z, 0, 15), z)
    return {"scales": sc.reshape(n, k // case["group"]), "values": (sc * (q - z)).reshape(n, k)}
