"""The low-bit path of a transformer layer, as it is measured: the residual's addition with the RMS norm and an 8-bit output,
rows brought to 8 bits without a norm, products with 4-bit weights for a few tokens, and the product of 8-bit rows and
8-bit weights.  `run` computes a case in plain torch operations, or, with `own` true, calls dtas_b200.ops."""
import math

import torch

own = False

F16, F32, E4M3, I8 = torch.float16, torch.float32, torch.float8_e4m3fn, torch.int8
QMAX = {"e4m3": 448.0, "int8": 127.0}
DTYPES = {"f16": F16, "f32": F32, "e4m3": E4M3, "int8": I8}


def _norm(name, m, h, out, x="f16"):
    return {"name": name, "op": "add_rms_norm", "m": m, "h": h, "x": x, "out": out}


def _quant(name, m, h, out, x="f16"):
    return {"name": name, "op": "quantize", "m": m, "h": h, "x": x, "out": out}


def _w4(name, m, n, k, group, x="f16", zero=False, tail="none"):
    return {"name": name, "op": "gemv_w4", "m": m, "n": n, "k": k, "group": group, "x": x, "zero": zero, "tail": tail}


def _f8(name, m, n, k, tail="none"):
    return {"name": name, "op": "gemm_nt_f8", "m": m, "n": n, "k": k, "tail": tail}


def listed():
    return [
        # one token between two blocks of a layer
        _norm("norm_token", 1, 4096, "f16"),
        # a long prompt, the rows of the 8-bit projections behind it
        _norm("norm_prompt_e4m3", 8192, 4096, "e4m3"),
        # a short ragged prompt of an odd width, fp32 activations
        _norm("norm_ragged_e4m3", 255, 2561, "e4m3", x="f32"),
        # the wide rows before a down projection: a batch of decoding sequences, and a prompt
        _quant("quantize_batch", 16, 10240, "e4m3"),
        _quant("quantize_prompt", 2048, 11008, "e4m3"),
        # one token through a square projection: latency
        _w4("w4_token_square", 1, 4096, 4096, 128),
        # one token through an up projection with its bias and activation, fine groups
        _w4("w4_token_up_gelu", 1, 22016, 4096, 32, tail="gelu"),
        # sixteen sequences through a down projection with zero points and the residual
        _w4("w4_batch_down", 16, 4096, 11008, 128, zero=True, tail="res1"),
        # four drafted tokens through a vocabulary projection, 8-bit rows
        _w4("w4_draft_head_e4m3", 4, 50280, 2560, 64, x="e4m3"),
        # a batch of decoding sequences with 8-bit weights
        _f8("f8_batch", 16, 12288, 4096),
        # a ragged prompt through an up projection
        _f8("f8_ragged_up_gelu", 1000, 10240, 2560, tail="gelu"),
        # a long prompt through a down projection with the residual
        _f8("f8_prompt_down", 8192, 4096, 11008, tail="res1"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["add_rms_norm", "quantize", "gemv_w4", "gemv_w4", "gemm_nt_f8"])
    if op in ("add_rms_norm", "quantize"):
        m, h = _log(rng, 1, 8192), _log(rng, 64, 16384)
        if rng.random() < 0.7:
            h = h // 8 * 8
        out = rng.choice(["f16", "e4m3", "int8"] if op == "add_rms_norm" else ["e4m3", "int8"])
        return {"op": op, "m": m, "h": h, "x": rng.choice(["f16", "f16", "f32"]), "out": out}
    if op == "gemv_w4":
        group = rng.choice([32, 64, 128])
        return {"op": op, "m": _log(rng, 1, 16), "n": _log(rng, 64, 50280), "k": group * max(1, _log(rng, 256, 11008) // group),
                "group": group, "x": rng.choice(["f16", "f16", "e4m3", "int8"]), "zero": rng.random() < 0.4,
                "tail": rng.choice(["none", "none", "bias", "gelu", "res1"])}
    return {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 64, 22016) if rng.random() < 0.3 else max(64, _log(rng, 64, 4096) // 8 * 8),
            "k": 16 * max(1, _log(rng, 256, 11008) // 16), "tail": rng.choice(["none", "none", "bias", "gelu", "res1"])}


def work(case):
    if case["op"] in ("add_rms_norm", "quantize"):
        m, h = case["m"], case["h"]
        i, o = (2 if case["x"] == "f16" else 4), (2 if case["out"] == "f16" else 1)
        if case["op"] == "quantize":
            return {"bytes": m * h * (i + o) + 4 * m, "flops": 2 * m * h}
        return {"bytes": m * h * (3 * i + o) + 2 * h + (4 * m if o == 1 else 0), "flops": 5 * m * h}
    m, n, k = case["m"], case["n"], case["k"]
    tail = 2 * n * (case["tail"] in ("bias", "gelu")) + 2 * m * n * (case["tail"] == "res1")
    if case["op"] == "gemm_nt_f8":
        return {"bytes": m * k + n * k + 4 * (m + n) + 2 * m * n + tail, "flops": 2 * m * n * k}
    groups = k // case["group"]
    x = 2 * m * k if case["x"] == "f16" else m * k + 4 * m
    return {"bytes": x + n * k // 2 + n * groups * (3 if case["zero"] else 2) + 2 * m * n + tail, "flops": 2 * m * n * k}


def _rows8(y, kind):
    """Rows of real numbers as 8-bit values and one scale a row."""
    top = y.abs().amax(-1, keepdim=True)
    q = y * torch.where(top > 0, QMAX[kind] / top, torch.zeros_like(top))
    q = q.to(E4M3) if kind == "e4m3" else q.round().to(I8)
    return q, (top / QMAX[kind]).squeeze(-1).to(F32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s = {"case": case}
    m = case["m"]
    if case["op"] in ("add_rms_norm", "quantize"):
        h = case["h"]
        # activations with a few columns far above the rest, as residual streams have them
        s["x"] = (randn(m, h) * torch.where(randn(h) > 2.5, 8.0, 1.0)).to(DTYPES[case["x"]])
        s["out"] = torch.empty(m, h, dtype=DTYPES[case["out"]], device="cuda")
        s["scale"] = torch.empty(m, device="cuda") if case["out"] != "f16" else None
        if case["op"] == "add_rms_norm":
            s["res"] = (randn(m, h) * 2).to(DTYPES[case["x"]])
            s["weight"] = (1 + 0.1 * randn(h)).to(F16)
            s["res_out"] = torch.empty_like(s["res"])
        return s
    n, k = case["n"], case["k"]
    x = randn(m, k)
    if case["op"] == "gemm_nt_f8":
        s["x"], s["x_scale"] = _rows8(x, "e4m3")
        s["w"], s["w_scale"] = _rows8(randn(n, k) * 0.02, "e4m3")
    else:
        s["x"], s["x_scale"] = (x.to(F16), None) if case["x"] == "f16" else _rows8(x, case["x"])
        groups = k // case["group"]
        zero = torch.randint(5, 12, (n, groups), generator=g, device="cuda") if case["zero"] else torch.full((n, groups), 8, device="cuda")
        codes = (randn(n, groups, case["group"]) * 2.7 + zero[:, :, None]).round_().clamp_(0, 15).to(torch.uint8).view(n, k)
        s["w"] = codes[:, 0::2] | (codes[:, 1::2] << 4)
        s["w_scale"] = (0.0075 * torch.exp(0.2 * randn(n, groups))).to(F16)
        s["w_zero"] = zero.to(torch.uint8) if case["zero"] else None
    s["bias"] = (0.1 * randn(n)).to(F16) if case["tail"] in ("bias", "gelu") else None
    s["res1"] = randn(m, n).to(F16) if case["tail"] == "res1" else None
    s["act"] = "gelu" if case["tail"] == "gelu" else None
    s["out"] = torch.empty(m, n, dtype=F16, device="cuda")
    return s


def _values(case, q, scale):
    """An 8-bit result as it is given back: e4m3 values as they are, whole numbers as the values that they stand for."""
    return [q if case["out"] == "e4m3" else (q * scale[:, None]).to(F16), scale]


def _tail(s, y):
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["act"] == "gelu":
        y = y * (0.5 + 0.5 * torch.erf(y * math.sqrt(0.5)))
    return y if s["res1"] is None else y + s["res1"]


def _plain(s):
    case, x = s["case"], s["x"].to(F32)
    if case["op"] == "add_rms_norm":
        h = x + s["res"].to(F32)
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * s["weight"].to(F32)
        if case["out"] == "f16":
            return [y.to(F16), h.to(s["res"].dtype)]
        return _values(case, *_rows8(y, case["out"])) + [h.to(s["res"].dtype)]
    if case["op"] == "quantize":
        return _values(case, *_rows8(x, case["out"]))
    if case["op"] == "gemm_nt_f8":
        y = (x @ s["w"].to(F32).t()) * s["x_scale"][:, None] * s["w_scale"]
        return _tail(s, y).to(F16)
    n, k, group = case["n"], case["k"], case["group"]
    w = torch.stack((s["w"] & 15, s["w"] >> 4), -1).view(n, k // group, group).to(F32)
    w = (w - (8 if s["w_zero"] is None else s["w_zero"].to(F32)[:, :, None])) * s["w_scale"].to(F32)[:, :, None]
    y = x @ w.view(n, k).t()
    if s["x_scale"] is not None:
        y = y * s["x_scale"][:, None]
    return _tail(s, y).to(F16)


def _own(s):
    from dtas_b200 import ops
    case = s["case"]
    if case["op"] == "add_rms_norm":
        ops.add_rms_norm(s["x"], s["res"], s["weight"], s["out"], res_out=s["res_out"], scale=s["scale"], eps=1e-6)
        return ([s["out"]] if case["out"] == "f16" else _values(case, s["out"], s["scale"])) + [s["res_out"]]
    if case["op"] == "quantize":
        ops.quantize(s["x"], s["out"], s["scale"])
        return _values(case, s["out"], s["scale"])
    if case["op"] == "gemm_nt_f8":
        return ops.gemm_nt_f8(s["x"], s["w"], s["x_scale"], s["w_scale"], s["out"], bias=s["bias"], res1=s["res1"], act=s["act"])
    return ops.gemv_w4(s["x"], s["w"], s["w_scale"], s["out"], w_zero=s["w_zero"], x_scale=s["x_scale"], bias=s["bias"],
                       res1=s["res1"], act=s["act"])


def run(state):
    return _own(state) if own else _plain(state)


def _exact8(y, kind):
    big = y.abs().max(-1, keepdim=True).values
    unit = (big / QMAX[kind]).clamp(min=1e-300)
    q = y / unit
    q = q.to(E4M3) if kind == "e4m3" else torch.round(q) * unit
    return [q, unit[:, 0]]


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "quantize":
        return _exact8(x, case["out"])
    if case["op"] == "add_rms_norm":
        h = x + s["res"].double()
        rms = torch.sqrt((h * h).sum(-1) / case["h"] + 1e-6)
        y = s["weight"].double() * h / rms[:, None]
        return ([y] if case["out"] == "f16" else _exact8(y, case["out"])) + [h]
    if s["x_scale"] is not None:
        x = x * s["x_scale"].double()[:, None]
    if case["op"] == "gemm_nt_f8":
        w = s["w"].double() * s["w_scale"].double()[:, None]
    else:
        w = torch.empty(case["n"], case["k"], dtype=torch.float64, device="cuda")
        w[:, 0::2] = (s["w"] % 16).double()
        w[:, 1::2] = (s["w"] // 16).double()
        for j in range(case["k"] // case["group"]):
            part = w[:, j * case["group"]:(j + 1) * case["group"]]
            part -= 8.0 if s["w_zero"] is None else s["w_zero"][:, j:j + 1].double()
            part *= s["w_scale"][:, j:j + 1].double()
    y = torch.mm(x, w.T)
    if s["bias"] is not None:
        y += s["bias"].double()
    if s["act"] == "gelu":
        y = 0.5 * y * torch.erfc(-y / math.sqrt(2.0))
    if s["res1"] is not None:
        y += s["res1"].double()
    return y
