"""Cases of the microscaled 4-bit operators and of rotary positions: inputs, the plain form of each operator, the
framework's call, the definition in 64 bits, and the work a pass cannot do without.

``own = False`` runs elementary torch operations, ``own = True`` the calls of ``feather_b200``.
"""
import math

import torch

own = False

DEVICE = "cuda"
BLOCK = 32  # elements that share a scale
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # one token's hidden state, as a projection leaves it, packed for the next product
        {"name": "pack 1x2048 fp32", "op": "pack", "rows": 1, "n": 2048, "dtype": "fp32"},
        # a large weight matrix, packed once when it is loaded
        {"name": "pack 16384x8192 fp16", "op": "pack", "rows": 16384, "n": 8192, "dtype": "fp16"},
        # a key projection's weights back in half precision
        {"name": "unpack 256x2048 fp16", "op": "unpack", "rows": 256, "n": 2048, "dtype": "fp16"},
        # a weight matrix back in FP32, for a check or another library
        {"name": "unpack 8192x8192 fp32", "op": "unpack", "rows": 8192, "n": 8192, "dtype": "fp32"},
        # key projection of one token: the smallest product, all latency
        {"name": "gemv 256x2048 bf16", "op": "gemv", "rows": 256, "n": 2048, "batch": 1, "vector": "bf16"},
        # odd sizes, rows that end inside a block, a few packed vectors at once
        {"name": "gemv 4099x5000 4 packed", "op": "gemv", "rows": 4099, "n": 5000, "batch": 4, "vector": "mxfp4"},
        # the framework's headline matrix at 4 bits
        {"name": "gemv 16384x16384 fp16", "op": "gemv", "rows": 16384, "n": 16384, "batch": 1, "vector": "fp16"},
        # a small batch of sequences through a down projection
        {"name": "gemm 2048x5632 33 rows", "op": "gemm", "rows": 2048, "n": 5632, "batch": 33, "out": "bf16"},
        # odd sizes throughout, FP32 result
        {"name": "gemm 5001x2050 200 rows", "op": "gemm", "rows": 5001, "n": 2050, "batch": 200, "out": "fp32"},
        # a prompt through a large projection
        {"name": "gemm 16384x8192 4096 rows", "op": "gemm", "rows": 16384, "n": 8192, "batch": 4096, "out": "bf16"},
        # queries and keys of one token far into a context, rotated and packed for the packed attention
        {"name": "rotary 1x36x64 packed", "op": "rotary", "tokens": 1, "heads": 36, "dim": 64, "rotated": 64,
         "layout": "half", "dtype": "fp32", "mode": "E5M2", "start": 100003, "base": 10000.0, "factor": 1.0},
        # a prompt's queries, half of each head rotated, positions scaled for a longer context
        {"name": "rotary 8192x32x128 fp16", "op": "rotary", "tokens": 8192, "heads": 32, "dim": 128, "rotated": 64,
         "layout": "interleaved", "dtype": "fp16", "mode": "", "start": 0, "base": 500000.0, "factor": 4.0},
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["pack", "unpack", "gemv", "gemv", "gemm", "gemm", "rotary"])
    if op in ("pack", "unpack"):
        n = _spread(rng, 1, 16384)
        rows = _spread(rng, 1, max(1, min(16384, 2 ** 26 // n)))
        if rng.random() < 0.5:
            n = -(-n // BLOCK) * BLOCK
        return {"op": op, "rows": rows, "n": n, "dtype": rng.choice(["fp16", "bf16", "fp32"])}
    if op == "gemv":
        rows, n = _spread(rng, 1, 32000), _spread(rng, 64, 16384)
        if rng.random() < 0.7:
            n = -(-n // 128) * 128
        return {"op": op, "rows": min(rows, 2 ** 28 // n), "n": n, "batch": rng.choice([1, 1, 1, 2, 3, 5, 8, 11]),
                "vector": rng.choice(["fp16", "bf16", "fp32", "mxfp4"])}
    if op == "gemm":
        rows, n, batch = _spread(rng, 32, 16384), _spread(rng, 64, 8192), _spread(rng, 1, 4096)
        if rng.random() < 0.7:
            n = -(-n // 128) * 128
        return {"op": op, "rows": rows, "n": n, "batch": batch, "out": rng.choice(["fp32", "bf16", "bf16", "fp16"])}
    dim = rng.choice([32, 64, 80, 96, 128, 256])
    heads = rng.randint(1, 40)
    return {"op": op, "tokens": _spread(rng, 1, max(1, 2 ** 25 // (heads * dim))), "heads": heads, "dim": dim,
            "rotated": dim if rng.random() < 0.6 else dim // 2, "layout": rng.choice(["half", "interleaved"]),
            "dtype": rng.choice(["fp16", "bf16", "fp32"]), "mode": rng.choice(["", "", "E5M2", "E4M3"]),
            "start": _spread(rng, 1, 1 << 20), "base": rng.choice([10000.0, 500000.0]), "factor": rng.choice([1.0, 4.0, 8.0])}


def _values(gen, *shape):
    """Normal values whose columns differ in size, a few of them by much, as activations and weights have them."""
    column = torch.exp(0.5 * torch.randn(shape[-1], generator=gen, device=DEVICE))
    column[:: 97] *= 16.0
    return torch.randn(*shape, generator=gen, device=DEVICE).mul_(column)


def _quantise(x):
    """(codes, two to a byte with the even element low; scale bytes) of the rows of x, plainly."""
    rows, n = x.shape
    blocks = -(-n // BLOCK)
    x = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - n)).view(rows, blocks, BLOCK)
    top = x.abs().amax(-1)
    exponent = (torch.frexp(top).exponent - 3).clamp(-127, 127)
    exponent = torch.where(top > 0, exponent, -127)
    y = torch.ldexp(x, -exponent[..., None])
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75).to(torch.uint8) + (a > 1.25).to(torch.uint8) + (a >= 1.75).to(torch.uint8)
            + (a > 2.5).to(torch.uint8) + (a >= 3.5).to(torch.uint8) + (a > 5.0).to(torch.uint8))
    code = code + 8 * torch.signbit(x).to(torch.uint8)
    fine = torch.isfinite(top)
    code = (code * fine[..., None].to(torch.uint8)).view(rows, blocks * BLOCK)
    scale = torch.where(fine, exponent + 127, 255).to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), scale


def _scale_values(scales):
    e = scales.to(torch.int32)
    return torch.where(e == 255, math.nan, torch.ldexp(torch.ones_like(e, dtype=torch.float32), e - 127))


def _dequantise(codes, scales, n):
    """The FP32 values of the rows, plainly."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1, BLOCK)
    return (table[c.int()] * _scale_values(scales)[..., None]).view(codes.shape[0], -1)[:, :n]


def _frequencies(case):
    """64-bit inverse frequencies, the positions' scale divided out of them."""
    i = torch.arange(0, case["rotated"], 2, dtype=torch.float64)
    return (case["base"] ** (-i / case["rotated"]) / case["factor"]).to(DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    op = case["op"]
    if op == "pack":
        return {"case": case, "x": _values(gen, case["rows"], case["n"]).to(DTYPES[case["dtype"]])}
    if op == "unpack":
        codes, scales = _quantise(_values(gen, case["rows"], case["n"]))
        return {"case": case, "codes": codes, "scales": scales}
    if op == "rotary":
        x = torch.randn(case["tokens"], case["heads"], case["dim"], generator=gen, device=DEVICE).to(DTYPES[case["dtype"]])
        return {"case": case, "x": x, "inv_freq": _frequencies(case),
                "positions": torch.arange(case["start"], case["start"] + case["tokens"], device=DEVICE)}
    codes, scales = _quantise(_values(gen, case["rows"], case["n"]).mul_(0.02))
    v = _values(gen, case["batch"], case["n"])
    if op == "gemv" and case["vector"] != "mxfp4":
        return {"case": case, "codes": codes, "scales": scales, "v": v.to(DTYPES[case["vector"]]), "v_scales": None}
    v, v_scales = _quantise(v)
    return {"case": case, "codes": codes, "scales": scales, "v": v, "v_scales": v_scales}


def _rotate(s, wide):
    """The rotated heads in the width `wide`, angles in 64 bits."""
    case, x = s["case"], s["x"].to(wide)
    r = case["rotated"]
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = torch.cos(angle).to(wide)[:, None, :], torch.sin(angle).to(wide)[:, None, :]
    if case["layout"] == "half":
        a, b = x[..., : r // 2], x[..., r // 2: r]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((turned, x[..., r:]), -1)


def _plain(s):
    case = s["case"]
    n = case.get("n")
    if case["op"] == "pack":
        codes, scales = _quantise(s["x"])
        return {"values": _dequantise(codes, scales, n).to(torch.bfloat16), "scales": scales.view(torch.float8_e8m0fnu)}
    if case["op"] == "unpack":
        return _dequantise(s["codes"], s["scales"], n).to(DTYPES[case["dtype"]])
    if case["op"] == "rotary":
        y = _rotate(s, torch.float32)
        if case["mode"]:
            return y.transpose(0, 1).contiguous().to(torch.float8_e5m2 if case["mode"] == "E5M2" else torch.float8_e4m3fn)
        return y.to(s["x"].dtype)
    v = s["v"].float() if s["v_scales"] is None else _dequantise(s["v"], s["v_scales"], n)
    y = v @ _dequantise(s["codes"], s["scales"], n).T
    return y if case["op"] == "gemv" else y.to(DTYPES[case["out"]])


def run(state):
    if not own:
        return _plain(state)
    import feather_b200 as fb
    case = state["case"]
    op = case["op"]
    if op == "pack":
        codes, scales = fb.pack_mxfp4_tensor(state["x"])
        # what is held in 4 bits, as the values it stands for: BF16 holds them all
        return {"values": fb.unpack_mxfp4_tensor(codes, scales, case["n"], torch.bfloat16), "scales": scales.view(torch.float8_e8m0fnu)}
    if op == "unpack":
        return fb.unpack_mxfp4_tensor(state["codes"], state["scales"], case["n"], DTYPES[case["dtype"]])
    if op == "rotary":
        y = fb.rotary_gpu(state["x"], state["positions"], state["inv_freq"], layout=case["layout"], mode=case["mode"] or None)
        if case["mode"]:
            return y.as_subclass(torch.Tensor).view(torch.float8_e5m2 if case["mode"] == "E5M2" else torch.float8_e4m3fn)
        return y
    shape = (case["rows"], case["n"])
    if op == "gemv":
        return fb.gemv_mxfp4_acc_fp32_gpu(state["codes"], state["scales"], state["v"], shape, v_scales=state["v_scales"])
    return fb.gemm_mxfp4_acc_fp32_gpu(state["codes"], state["scales"], state["v"], state["v_scales"], shape, out_dtype=DTYPES[case["out"]])


def work(case):
    op = case["op"]
    if op == "rotary":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": n * (SIZE[case["dtype"]] + (1 if case["mode"] else SIZE[case["dtype"]])) + 8 * (case["tokens"] + case["rotated"] // 2),
                "flops": 3 * case["tokens"] * case["heads"] * case["rotated"]}
    rows, n = case["rows"], case["n"]
    blocks = -(-n // BLOCK)
    packed = 17 * blocks  # bytes of one packed row
    if op == "pack":
        return {"bytes": rows * (n * (SIZE[case["dtype"]] + 2) + packed), "flops": 4 * rows * n}
    if op == "unpack":
        return {"bytes": rows * (packed + n * SIZE[case["dtype"]]), "flops": 2 * rows * n}
    batch = case["batch"]
    if op == "gemv":
        vector = packed if case["vector"] == "mxfp4" else n * SIZE[case["vector"]]
        return {"bytes": rows * packed + batch * (vector + 4 * rows), "flops": 2 * rows * n * batch}
    return {"bytes": (rows + batch) * packed + batch * rows * SIZE[case["out"]], "flops": 2 * rows * n * batch}


def _decode64(codes, scales, n):
    """The values from the format's definition: sign, two exponent bits of bias 1, one mantissa bit, times a power of two."""
    c = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.int32, device=codes.device)
    c[:, 0::2], c[:, 1::2] = codes.int() % 16, codes.int() // 16
    e, m = (c // 2) % 4, (c % 2).double()
    magnitude = torch.where(e == 0, m * 0.5, (1 + 0.5 * m) * torch.exp2((e - 1).double()))
    sign = 1.0 - 2.0 * (c // 8).double()
    scale = torch.exp2(scales.double() - 127.0)
    scale[scales == 255] = math.nan
    return (sign * magnitude * scale.repeat_interleave(BLOCK, 1))[:, :n]


def _exponent64(x):
    """floor(log2 |x|) of 64-bit values, from their exponent bits."""
    return ((x.double().contiguous().view(torch.int64) >> 52) & 2047) - 1023


def _on_grid64(x, mantissa, lowest):
    """x rounded to a format of so many mantissa bits and that lowest normal exponent, ties to even, in 64 bits."""
    step = torch.exp2((_exponent64(x).clamp(min=lowest) - mantissa).double())
    return torch.round(x / step) * step


def _nearest64(x):
    """(values, scales) of x on the grid of its blocks, in 64 bits: steps of a half below 2, of 1 below 4, of 2 above, ties to even."""
    rows, n = x.shape
    blocks = -(-n // BLOCK)
    x = torch.cat((x.double(), x.new_zeros(rows, blocks * BLOCK - n).double()), 1).view(rows, blocks, BLOCK)
    top = x.abs().amax(-1, keepdim=True)
    scale = torch.exp2((_exponent64(top) - 2).clamp(-127, 127).double())
    y = x / scale
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    values = (torch.round(y / step) * step).clamp(-6, 6) * scale
    return values.view(rows, -1)[:, :n], scale[..., 0]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pack":
        values, scales = _nearest64(s["x"])
        return {"values": values, "scales": scales}
    if case["op"] == "unpack":
        return _decode64(s["codes"], s["scales"], case["n"])
    if case["op"] == "rotary":
        # a rotation as a product of complex numbers
        x, r = s["x"].double(), case["rotated"]
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE), s["positions"].double()[:, None, None] * s["inv_freq"])
        z = torch.complex(x[..., : r // 2], x[..., r // 2: r]) if case["layout"] == "half" else torch.view_as_complex(x[..., :r].unflatten(-1, (-1, 2)).contiguous())
        z = z * turn
        x[..., :r] = torch.cat((z.real, z.imag), -1) if case["layout"] == "half" else torch.view_as_real(z).flatten(-2)
        if case["mode"]:
            x = x.transpose(0, 1).contiguous()
            return _on_grid64(x, 2, -14) if case["mode"] == "E5M2" else _on_grid64(x, 3, -6)
        return x
    v = s["v"].double() if s["v_scales"] is None else _decode64(s["v"], s["v_scales"], case["n"])
    return v @ _decode64(s["codes"], s["scales"], case["n"]).T
