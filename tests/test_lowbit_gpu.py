"""The low-bit path on the GPU against plain 64-bit restatements of its formulas.

Tolerances count roundings.  fp32 arithmetic in front of the last rounding: a row sum of n terms is added in chains of at most
32 terms and two trees of five levels, 42 roundings of 2^-24, half of that on its root, plus six further operations: under
32 * 2^-24 = 2^-19 of the value.  The last rounding is half a step of the stored type: fp16 2^-11 of the value (2^-25 below the normal
range), e4m3 2^-4 (2^-10 of the scale below the normal range), int8 half the scale."""
import math

import pytest
import torch

from dtas_b200 import _abi, ops, weights

pytestmark = pytest.mark.gpu

F16, F32, I8, E4M3 = torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn
Q = {I8: 127.0, E4M3: 448.0}
FP32 = 2.0 ** -19


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=gen(seed), device="cuda") * scale


def assert_fp16_close(got, want, slack, what=""):
    """got (fp16, or fp32 holding an fp16 value) within half a step of fp16 and `slack` of the exact values; NaN where those are
    (a drawn e4m3 element beyond 464 is one), finite elsewhere."""
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan) and bool(torch.isfinite(got[~nan].float()).all()), what
    got, want, slack = got[~nan], want[~nan], slack[~nan] if torch.is_tensor(slack) and slack.dim() else slack
    err = (got.double() - want).abs()
    tol = (want.abs() + slack) * 2.0 ** -11 + slack + 2.0 ** -25
    bad = (err > tol).nonzero()[:, 0]
    assert len(bad) == 0, f"{what}: {len(bad)} of {got.numel()} off, the first {float(got[bad[0]])} for {float(want[bad[0]])}"


def assert_rows8(q, scale, y, what=""):
    """q and scale are the 8-bit form of the rows y (fp64)."""
    top = y.abs().amax(-1)
    want_scale = top / Q[q.dtype]
    assert ((scale.double() - want_scale).abs() <= want_scale * FP32 + 1e-300).all(), what
    s = want_scale[:, None]
    half = 0.5 * s if q.dtype == I8 else (y.abs() * 2.0 ** -4).clamp(min=2.0 ** -10 * s)
    tol = half * (1 + 2.0 ** -10) + (top * 4 * FP32)[:, None]
    err = (q.double() * scale.double()[:, None] - y).abs()
    assert (err <= tol).all(), f"{what}: off by {(err / tol.clamp(min=1e-300)).max()} of what rounding explains"
    if q.dtype == I8:
        assert int(q.min()) >= -127


def norm_of(x, res, weight, eps):
    h = x.double() if res is None else x.double() + res.double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * weight.double()
    return h, y


def assert_h(got, h):
    tol = h.abs() * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25 if got.dtype == F16 else h.abs() * 2.0 ** -24 + 1e-44
    assert ((got.double() - h).abs() <= tol).all()


WIDTHS = [1, 7, 64, 100, 264, 1024, 2561, 4096, 8200, 11008, 16384, 16392, 20001, 32768, 32776, 70001]


@pytest.mark.parametrize("out_dtype", [F16, I8, E4M3])
@pytest.mark.parametrize("in_dtype", [F16, F32])
@pytest.mark.parametrize("h", WIDTHS)
def test_add_rms_norm(cuda_device, h, in_dtype, out_dtype):
    for m in (1, 5, 600 if h <= 4096 else 3):
        x, res = randn(m, h, seed=h + m).to(in_dtype), randn(m, h, seed=h + m + 1, scale=2).to(in_dtype)
        w = (1 + randn(h, seed=h + 2, scale=0.1)).to(F16)
        out = torch.empty(m, h, dtype=out_dtype, device="cuda")
        res_out, scale = torch.empty_like(x), torch.empty(m, device="cuda")
        assert ops.add_rms_norm(x, res, w, out, res_out=res_out, scale=scale) is out
        hh, y = norm_of(x, res, w, 1e-6)
        assert_h(res_out, hh)
        if out_dtype == F16:
            assert_fp16_close(out, y, y.abs().max() * FP32, f"m={m}")
        else:
            assert_rows8(out, scale, y, f"m={m}")


@pytest.mark.parametrize("out_dtype", [I8, E4M3])
@pytest.mark.parametrize("in_dtype", [F16, F32])
@pytest.mark.parametrize("h", WIDTHS)
def test_quantize(cuda_device, h, in_dtype, out_dtype):
    for m in (1, 6, 700 if h <= 4096 else 2):
        x = randn(m, h, seed=h + m, scale=3).to(in_dtype)
        q, scale = torch.empty(m, h, dtype=out_dtype, device="cuda"), torch.empty(m, device="cuda")
        ops.quantize(x, q, scale)
        assert_rows8(q, scale, x.double(), f"m={m}")


@pytest.mark.parametrize("h", [264, 257, 40000])
def test_norm_without_residual_and_in_place(cuda_device, h):
    m = 5
    x, res = randn(m, h, seed=1).to(F16), randn(m, h, seed=2).to(F16)
    w = (1 + randn(h, seed=3, scale=0.1)).to(F16)
    # no residual: the norm of x itself, in 8 bits too
    q, scale = torch.empty(m, h, dtype=I8, device="cuda"), torch.empty(m, device="cuda")
    ops.add_rms_norm(x, None, w, q, scale=scale, eps=1e-3)
    assert_rows8(q, scale, norm_of(x, None, w, 1e-3)[1])
    # the residual stream updated in place, and the result written over x
    hh, y = norm_of(x, res, w, 1e-6)
    ops.add_rms_norm(x, res, w, x, res_out=res)
    assert_h(res, hh)
    assert_fp16_close(x, y, y.abs().max() * FP32)


@pytest.mark.parametrize("op,m,h,in_dtype", [("norm", 40001, 64, F16), ("norm", 5003, 1000, F16), ("norm", 900, 4104, F16),
                                             ("norm", 300, 16384, F16), ("norm", 1500, 8191, F16), ("norm", 601, 16383, F16),
                                             ("norm", 1003, 4361, F16), ("quantize", 12001, 136, F16),
                                             ("quantize", 12001, 1024, F32), ("quantize", 20003, 8, F16)])
def test_more_rows_than_fit_at_once(cuda_device, op, m, h, in_dtype):
    assert _abi.variant_of("add_rms_norm" if op == "norm" else op, m, h).endswith("_stream")
    x, res = randn(m, h, seed=m).to(in_dtype), randn(m, h, seed=m + 1, scale=2).to(in_dtype)
    x[m // 2], res[m // 2] = 0, 0
    x[m - 1, h - 1] = math.nan
    w = (1 + randn(h, seed=2, scale=0.1)).to(F16)
    fine = torch.arange(m - 1, device="cuda")
    for out_dtype in (I8, E4M3) + ((F16,) if op == "norm" else ()):
        out = torch.empty(m, h, dtype=out_dtype, device="cuda")
        scale = torch.full((m,), 7.0, device="cuda")
        if op == "quantize":
            y = x.double()
            ops.quantize(x, out, scale)
        else:
            hh, y = norm_of(x, res, w, 1e-6)
            stream = res.clone()
            ops.add_rms_norm(x, stream, w, out, res_out=stream, scale=scale)      # the residual stream updated in place
            assert_h(stream[fine], hh[fine])
            plain = torch.empty_like(out)                                          # neither a residual nor its sum
            ops.add_rms_norm(x, None, w, plain, scale=torch.empty_like(scale))
            one = torch.empty_like(out)
            ops.add_rms_norm(x, torch.zeros_like(x), w, one, scale=torch.empty_like(scale))
            assert torch.equal(plain.view(torch.uint8), one.view(torch.uint8))
        if out_dtype == F16:
            assert_fp16_close(out[fine], y[fine], y[fine].abs().max() * FP32)
            assert torch.isnan(out[m - 1]).all()
        else:
            assert_rows8(out[fine], scale[fine], y[fine])
            assert scale[m // 2] == 0 and torch.isnan(scale[m - 1])


@pytest.mark.parametrize("in_dtype,out_dtype", [(F16, I8), (F16, E4M3), (F32, I8), (F32, E4M3)])
@pytest.mark.parametrize("h", [64, 65, 40000])
def test_rows_of_zeros_infinities_and_tiny_values(cuda_device, h, in_dtype, out_dtype):
    x = randn(6, h, seed=h).to(in_dtype)
    x[1] = 0
    x[2, h // 2] = math.inf
    x[3, h // 3] = math.nan
    tiny = 1e-38 if in_dtype == F32 else 6e-8        # below 1 / FLT_MAX times 448 in fp32: Q / max overflows
    x[4] = tiny * (1 + torch.arange(h, device="cuda") % 3)
    x[5, 0] = 60000
    q, scale = torch.empty(6, h, dtype=out_dtype, device="cuda"), torch.full((6,), 7.0, device="cuda")
    ops.quantize(x, q, scale)
    keep = [0, 5] if in_dtype == F32 else [0, 4, 5]
    assert_rows8(q[keep], scale[keep], x[keep].double())
    assert scale[1] == 0 and (q[1].float() == 0).all()
    assert torch.isnan(scale[2]) and torch.isnan(scale[3])
    # scale of the tiny row is a subnormal number (granularity 2^-149), the values over it are not
    want = x[4].double() / x[4].double().abs().max() * Q[out_dtype]
    step = 0.5 if out_dtype == I8 else want * 2.0 ** -4
    assert ((q[4].double() - want).abs() <= step * (1 + 2.0 ** -10) + 1e-3).all()
    # the same rows through the norm: NaN rows stay NaN, zero rows stay zero, no other row is touched by them
    w = (1 + randn(h, seed=3, scale=0.1)).to(F16)
    ops.add_rms_norm(x, None, w, q, scale=scale)
    _, y = norm_of(x, None, w, 1e-6)
    assert_rows8(q[[0, 5]], scale[[0, 5]], y[[0, 5]])
    assert scale[1] == 0 and (q[1].float() == 0).all() and torch.isnan(scale[2]) and torch.isnan(scale[3])
    out = torch.empty(6, h, dtype=F16, device="cuda")
    ops.add_rms_norm(x, None, w, out)
    assert torch.isnan(out[3]).all() and (out[1] == 0).all() and torch.isfinite(out[[0, 1, 4, 5]].float()).all()


def _offset(t, by):
    """A contiguous copy of t that starts `by` elements behind an allocation's start, and the buffer it lies in."""
    buf = torch.zeros(t.numel() + by + 64, dtype=t.dtype, device=t.device)
    view = buf[by:by + t.numel()].view(t.shape)
    view.copy_(t)
    return view


@pytest.mark.parametrize("off", [1, 3])
def test_rows_at_odd_addresses(cuda_device, off):
    m, h = 9, 512
    x, res, w = randn(m, h, seed=1).to(F16), randn(m, h, seed=2).to(F16), (1 + randn(h, seed=3, scale=0.1)).to(F16)
    hh, y = norm_of(x, res, w, 1e-6)
    for which in range(4):
        xs, rs, ws = (_offset(t, off) if which == i else t for i, t in enumerate((x, res, w)))
        buf = torch.zeros(m * h + 64, dtype=E4M3, device="cuda")
        q = buf[off if which == 3 else 0:][:m * h].view(m, h)
        scale, ro = torch.empty(m, device="cuda"), torch.empty_like(x)
        ops.add_rms_norm(xs, rs, ws, q, res_out=ro, scale=scale)
        assert_h(ro, hh)
        assert_rows8(q, scale, y)
        assert (buf[(off if which == 3 else 0) + m * h:].float() == 0).all() and (which != 3 or (buf[:off].float() == 0).all())


# ---- 4-bit products ---------------------------------------------------------------------------------
def w4_case(m, n, k, group, x_dtype=F16, zero=False, seed=0):
    groups = k // group
    c = {"codes": torch.randint(0, 16, (n, k), generator=gen(seed), device="cuda", dtype=torch.uint8)}
    c["w"] = weights.pack_w4(c["codes"])
    c["w_scale"] = (0.01 * torch.exp(0.3 * randn(n, groups, seed=seed + 1))).to(F16)
    c["w_zero"] = torch.randint(0, 16, (n, groups), generator=gen(seed + 2), device="cuda", dtype=torch.uint8) if zero else None
    x = randn(m, k, seed=seed + 3)
    if x_dtype == F16:
        c["x"], c["x_scale"] = x.to(F16), None
    else:
        c["x"] = (x * 40).round().clamp(-127, 127).to(I8) if x_dtype == I8 else (x * 100).to(E4M3)
        c["x_scale"] = 0.01 + 0.01 * torch.rand(m, generator=gen(seed + 4), device="cuda")
    z = 8.0 if c["w_zero"] is None else c["w_zero"].double()[..., None]
    w = ((c["codes"].double().view(n, groups, group) - z) * c["w_scale"].double()[..., None]).view(n, k)
    xs = c["x"].double() if c["x_scale"] is None else c["x"].double() * c["x_scale"].double()[:, None]
    c["y"] = xs @ w.t()
    # codes (up to 15) and zero points times the group's sum of x are added up apart, so what is rounded is measured by 30
    # times the scale times |x|; products are exact; sums of a group inside the MMAs (a truncated step of 2^-23 each), one
    # fp32 rounding a group and warp, the scales: that many steps of 2^-23, at most
    mag = xs.abs() @ (30 * c["w_scale"].double()[..., None].expand(n, groups, group).reshape(n, k)).t()
    c["slack"] = mag * ((max(group // 16, k // 32) + k // group + 24) * 2.0 ** -23)
    return c


def w4_call(c, out, **kw):
    return ops.gemv_w4(c["x"], c["w"], c["w_scale"], out, w_zero=c["w_zero"], x_scale=c["x_scale"], **kw)


FAST = [(32, 32), (64, 64), (64, 32), (128, 128), (160, 32), (192, 64), (192, 96), (192, 192), (1056, 32), (1280, 128), (2560, 64),
        (4096, 128), (4096, 4096), (11008, 128), (10240, 32)]
SLOW = [(2, 1), (2, 2), (30, 10), (34, 17), (48, 16), (100, 50), (1000, 40)]


@pytest.mark.parametrize("x_dtype", [F16, I8, E4M3])
@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("k,group", FAST + SLOW)
def test_gemv_w4(cuda_device, k, group, zero, x_dtype):
    for m, n in ((1, 100), (2, 1), (7, 17), (8, 33), (9, 48), (16, 15)):
        c = w4_case(m, n, k, group, x_dtype, zero, seed=k + m)
        buf = torch.full((m * n + 64,), 3.0, dtype=F16, device="cuda")
        w4_call(c, buf[:m * n].view(m, n))
        assert_fp16_close(buf[:m * n].view(m, n), c["y"], c["slack"], f"m={m} n={n}")
        assert (buf[m * n:] == 3.0).all()


@pytest.mark.parametrize("m", [1, 3, 16])
@pytest.mark.parametrize("n,k,group", [(4096, 4096, 128), (4097, 2560, 32), (50280, 256, 64)])
def test_gemv_w4_wide(cuda_device, m, n, k, group):
    c = w4_case(m, n, k, group, seed=n)
    out = torch.empty(m, n, dtype=F16, device="cuda")
    w4_call(c, out)
    assert_fp16_close(out, c["y"], c["slack"])
    again = torch.empty_like(out)
    w4_call(c, again)
    assert torch.equal(out, again)      # the same sums in the same order


@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("x_dtype", [F16, I8])
@pytest.mark.parametrize("m,n,k,group", [(16, 4096, 11008, 128), (16, 9001, 20480, 64), (8, 5000, 16384, 32), (9, 9000, 4096, 128), (2, 300, 40960, 256)])
def test_gemv_w4_with_k_shared_out(cuda_device, m, n, k, group, x_dtype, zero):
    """Rows of x that do not fit one CTA's shared memory: K over the CTAs of a cluster, several tiles each, in one
    batch and in several."""
    c = w4_case(m, n, k, group, x_dtype, zero, seed=k)
    out = torch.empty(m, n, dtype=F16, device="cuda")
    bias = randn(n, seed=5).to(F16)
    w4_call(c, out, bias=bias)
    ops.poll_status()
    assert_fp16_close(out, c["y"] + bias.double(), c["slack"])
    again = torch.empty_like(out)
    w4_call(c, again, bias=bias)
    assert torch.equal(out, again)


def gelu(v):
    return v * (0.5 + 0.5 * torch.erf(v * math.sqrt(0.5)))


@pytest.mark.parametrize("k,group", [(256, 32), (60, 30)])
@pytest.mark.parametrize("out_dtype", [F16, F32])
@pytest.mark.parametrize("m", [1, 5, 16])
def test_gemv_w4_tails(cuda_device, m, out_dtype, k, group):
    n = 77
    c = w4_case(m, n, k, group, zero=True, seed=m)
    bias, r1, r2 = randn(n, seed=5).to(F16), randn(m, n, seed=6).to(F16), randn(m, n, seed=7).to(F16)
    b, d1, d2 = bias.double(), r1.double(), r2.double()
    for kw, want in (({"bias": bias}, c["y"] + b), ({"act": "gelu"}, gelu(c["y"])), ({"bias": bias, "act": "gelu", "res1": r1}, gelu(c["y"] + b) + d1),
                     ({"res1": r1, "res2": r2}, c["y"] + d1 + d2)):
        out = torch.empty(m, n, dtype=out_dtype, device="cuda")
        w4_call(c, out, **kw)
        # gelu's slope is under 1.13 and its erf is good to 5e-7 of the argument
        terms = c["y"].abs() + b.abs() + d1.abs() + d2.abs()
        assert_fp16_close(out, want, 1.13 * c["slack"] + terms * (2.0 ** -20), str(list(kw)))
        assert out_dtype == F16 or torch.equal(out, out.half().float())


def test_gemv_w4_at_odd_addresses(cuda_device):
    c = w4_case(3, 40, 128, 32, seed=9)
    for key, by in (("x", 1), ("w", 1), ("w", 8), ("x", 4)):
        d = dict(c)
        d[key] = _offset(c[key], by)
        out = torch.empty(3, 40, dtype=F16, device="cuda")
        w4_call(d, out)
        assert_fp16_close(out, c["y"], c["slack"], f"{key} + {by}")
    out = _offset(torch.empty(3, 40, dtype=F16, device="cuda"), 1)
    w4_call(c, out)
    assert_fp16_close(out, c["y"], c["slack"])


@pytest.mark.parametrize("k", [128, 60])
def test_gemv_w4_keeps_infinities_to_their_rows(cuda_device, k):
    c = w4_case(4, 24, k, k // 2, seed=3)
    c["x"][1, 5] = math.inf
    c["x"][2, 7] = math.nan
    c["w_scale"][11, 0] = math.inf
    out = torch.empty(4, 24, dtype=F16, device="cuda")
    w4_call(c, out)
    plain = [n for n in range(24) if n != 11]
    for i in (0, 3):
        assert torch.isfinite(out[i, plain].float()).all()
        assert_fp16_close(out[i, plain], c["y"][i, plain], c["slack"][i, plain])
    assert torch.isnan(out[2]).all() and not torch.isfinite(out[1].float()).any() and not torch.isfinite(out[:, 11].float()).any()


def test_weights_of_four_bits_reach_the_product(cuda_device):
    w = randn(96, 256, seed=1, scale=0.05)
    for zp in (False, True):
        codes, scale, zero = weights.quantize_w4(w, 64, zp)
        wd = weights.dequantize_w4(codes, scale, zero, dtype=F32).double()
        x = randn(2, 256, seed=2).to(F16)
        out = torch.empty(2, 96, dtype=F16, device="cuda")
        ops.gemv_w4(x, codes, scale, out, w_zero=zero)
        assert_fp16_close(out, x.double() @ wd.t(), x.double().abs() @ wd.abs().t() * (40 * 2.0 ** -22))


# ---- products of 8-bit operands ------------------------------------------------------------------------
def f8_case(m, n, k, seed=0):
    c = {"x": randn(m, k, seed=seed, scale=60).to(E4M3), "w": randn(n, k, seed=seed + 1, scale=60).to(E4M3),
         "x_scale": 0.01 * (0.5 + torch.rand(m, generator=gen(seed + 2), device="cuda")),
         "w_scale": 0.001 * (0.5 + torch.rand(n, generator=gen(seed + 3), device="cuda"))}
    s = c["x_scale"].double()[:, None] * c["w_scale"].double()
    c["y"], c["abs"] = (c["x"].double() @ c["w"].double().t()) * s, (c["x"].double().abs() @ c["w"].double().abs().t()) * s
    # e4m3 products are exact; one accumulation step in fp32 per MMA of 32 k and the joins of split sums
    c["slack"] = c["abs"] * ((k // 32 + 40) * 2.0 ** -22)
    return c


def f8_call(c, out, **kw):
    ops.gemm_nt_f8(c["x"], c["w"], c["x_scale"], c["w_scale"], out, **kw)
    ops.poll_status()
    return out


@pytest.mark.parametrize("n,k", [(1, 16), (17, 48), (128, 128), (130, 1040), (1000, 144), (512, 4096), (1, 7), (33, 40), (260, 8192)])
@pytest.mark.parametrize("m", [1, 5, 16, 33, 64, 65, 128, 129, 255, 300, 1025])
def test_gemm_f8(cuda_device, m, n, k):
    c = f8_case(m, n, k, seed=m + n + k)
    buf = torch.full((m * n + 64,), 3.0, dtype=F16, device="cuda")
    f8_call(c, buf[:m * n].view(m, n))
    assert_fp16_close(buf[:m * n].view(m, n), c["y"], c["slack"])
    assert (buf[m * n:] == 3.0).all()


CODES = [(64, 1), (128, 1), (256, 1), (64, 3), (128, 2), (256, 2), (512, 1), (513, 1), (4096 + 64, 0), (4096 + 128, 0), (8192 + 64, 0), (8192 + 128, 0)]
SMALL_CODES = [(1024, 1), (1024, 3), (2048, 0), (16384 + 2, 0), (16384 + 3, 0), (16384 + 4, 0)]


@pytest.mark.parametrize("tail", ["none", "gelu", "res"])
@pytest.mark.parametrize("m,code", [(m, c) for m in (200, 333) for c in CODES] + [(m, c) for m in (1, 20, 50) for c in SMALL_CODES])
def test_gemm_f8_in_every_kernel(cuda_device, m, code, tail):
    n, k = 328, 1600
    c = f8_case(m, n, k, seed=m)
    r1 = randn(m, n, seed=6).to(F16)
    bias = randn(n, seed=7).to(F16)
    kw, want = {"none": ({}, c["y"]), "gelu": ({"bias": bias, "act": "gelu"}, gelu(c["y"] + bias.double())), "res": ({"res1": r1}, c["y"] + r1.double())}[tail]
    lib = _abi.lib()
    _abi.check(lib.dtas_gemm_set_override(*code))
    try:
        for dt in (F16, F32):
            out = f8_call(c, torch.empty(m, n, dtype=dt, device="cuda"), **kw)
            assert_fp16_close(out, want, 1.13 * c["slack"] + (c["y"].abs() + 8) * 2.0 ** -20, f"{dt}")
    finally:
        lib.dtas_gemm_set_override(0, 0)


@pytest.mark.parametrize("m", [3, 300])
def test_gemm_f8_into_a_slab_and_at_odd_addresses(cuda_device, m):
    n, k = 100, 256
    c = f8_case(m, n, k, seed=4)
    wide = torch.full((m, 3 * n), 5.0, dtype=F16, device="cuda")
    f8_call(c, wide[:, n:2 * n])
    assert_fp16_close(wide[:, n:2 * n], c["y"], c["slack"])
    assert (wide[:, :n] == 5.0).all() and (wide[:, 2 * n:] == 5.0).all()
    for key in ("x", "w", "x_scale", "w_scale"):
        d = dict(c)
        d[key] = _offset(c[key], 1)
        assert_fp16_close(f8_call(d, torch.empty(m, n, dtype=F16, device="cuda")), c["y"], c["slack"], key)


@pytest.mark.parametrize("m", [2, 150])
def test_gemm_f8_keeps_nan_to_its_row(cuda_device, m):
    c = f8_case(m, 64, 128, seed=8)
    c["x"][1, 3] = math.nan
    out = f8_call(c, torch.empty(m, 64, dtype=F16, device="cuda"))
    assert torch.isnan(out[1]).all()
    rest = [i for i in range(m) if i != 1]
    assert_fp16_close(out[rest], c["y"][rest], c["slack"][rest])


# ---- together, and as they are called -------------------------------------------------------------------
def test_refusals_leave_the_outputs_alone(cuda_device):
    x, w = randn(2, 64).to(F16), torch.ones(64, dtype=F16, device="cuda")
    q, s = torch.zeros(2, 64, dtype=I8, device="cuda"), torch.zeros(2, device="cuda")
    codes, ws = torch.zeros(8, 32, dtype=torch.uint8, device="cuda"), torch.ones(8, 2, dtype=F16, device="cuda")
    y = torch.zeros(2, 8, dtype=F16, device="cuda")
    x8, w8 = x.to(E4M3), torch.zeros(8, 64, device="cuda").to(E4M3)
    calls = [lambda: ops.add_rms_norm(x, x, w, q), lambda: ops.add_rms_norm(x, x.float(), w, q, scale=s), lambda: ops.add_rms_norm(x, x, w.float(), q, scale=s),
             lambda: ops.add_rms_norm(x, x[:1], w, q, scale=s), lambda: ops.add_rms_norm(x, x, w, q, scale=s[:1]), lambda: ops.add_rms_norm(x, x, w, q.float(), scale=s),
             lambda: ops.add_rms_norm(x.t(), x.t(), w, q, scale=s), lambda: ops.add_rms_norm(x, x, w, q, scale=s, res_out=x.float()),
             lambda: ops.quantize(x, x, s), lambda: ops.quantize(x, q, s.half()), lambda: ops.quantize(x.bfloat16(), q, s),
             lambda: ops.gemv_w4(x, codes, ws.float(), y), lambda: ops.gemv_w4(x, codes.char(), ws, y), lambda: ops.gemv_w4(x, codes, ws[:, :1].expand(8, 3), y),
             lambda: ops.gemv_w4(x, codes, ws, y, w_zero=codes), lambda: ops.gemv_w4(x, codes, ws, y, x_scale=s), lambda: ops.gemv_w4(q, codes, ws, y),
             lambda: ops.gemv_w4(x, codes, ws, y, bias=w[:7]), lambda: ops.gemv_w4(x, codes, ws, y, act="relu"), lambda: ops.gemv_w4(x.float(), codes, ws, y),
             lambda: ops.gemv_w4(randn(17, 64).to(F16), codes, ws, torch.empty(17, 8, dtype=F16, device="cuda")),
             lambda: ops.gemm_nt_f8(x, w8, s, ws[:, 0].float(), y), lambda: ops.gemm_nt_f8(x8, w8.to(F16), s, ws[:, 0].float(), y),
             lambda: ops.gemm_nt_f8(x8, w8, s, s, y), lambda: ops.gemm_nt_f8(x8, w8[:, :32], s, torch.ones(8, device="cuda"), y),
             lambda: ops.gemm_nt_f8(x8, w8, s, torch.ones(8), y)]
    for i, call in enumerate(calls):
        with pytest.raises(_abi.DtasError):
            call()
            pytest.fail(f"call {i} was not refused")
    assert (q == 0).all() and (s == 0).all() and (y == 0).all()


def mlp_weights(h, f, seed=50):
    w_up, w_down = randn(f, h, seed=seed, scale=0.05).to(F16), randn(h, f, seed=seed + 1, scale=0.05).to(F16)
    d = {"norm": (1 + randn(h, seed=seed + 2, scale=0.1)).to(F16), "bias": randn(f, seed=seed + 3, scale=0.1).to(F16)}
    for name, w in (("up", w_up), ("down", w_down)):
        q, s = torch.empty(w.shape, dtype=E4M3, device="cuda"), torch.empty(w.shape[0], device="cuda")
        d[name + "8"] = (ops.quantize(w, q, s), s)
        d[name + "4"] = weights.quantize_w4(w, 64, True)
    return d


class Mlp:
    """A feed-forward block as a layer would run it: residual + norm, up projection with GELU, down projection."""

    def __init__(self, d, m, h, f):
        self.d = d
        new = lambda *shape, dt=F16: torch.empty(*shape, dtype=dt, device="cuda")  # noqa: E731
        self.h8, self.hs, self.h16 = new(m, h, dt=E4M3), new(m, dt=F32), new(m, h)
        self.u, self.u8, self.us, self.y = new(m, f), new(m, f, dt=E4M3), new(m, dt=F32), new(m, h)

    def prompt(self, x, res):
        d = self.d
        ops.add_rms_norm(x, res, d["norm"], self.h8, res_out=res, scale=self.hs)
        ops.gemm_nt_f8(self.h8, d["up8"][0], self.hs, d["up8"][1], self.u, bias=d["bias"], act="gelu")
        ops.quantize(self.u, self.u8, self.us)
        return ops.gemm_nt_f8(self.u8, d["down8"][0], self.us, d["down8"][1], self.y, res1=res)

    def token(self, x, res):
        d = self.d
        ops.add_rms_norm(x, res, d["norm"], self.h8, res_out=res, scale=self.hs)
        ops.gemv_w4(self.h8, d["up4"][0], d["up4"][1], self.u, w_zero=d["up4"][2], x_scale=self.hs, bias=d["bias"], act="gelu")
        return ops.gemv_w4(self.u, d["down4"][0], d["down4"][1], self.y, w_zero=d["down4"][2], res1=res)


def mlp_plain(d, x, res, token, block):
    """The block in 64 bits, taking the 8-bit rows that the block wrote for what they stand for."""
    h = x.double() + res.double()
    rows = block.h8.double() * block.hs.double()[:, None]
    if token:
        up, down = (weights.dequantize_w4(*d[n + "4"], dtype=torch.float64) for n in ("up", "down"))
        u = block.u.double()
    else:
        up, down = (d[n + "8"][0].double() * d[n + "8"][1].double()[:, None] for n in ("up", "down"))
        u = block.u8.double() * block.us.double()[:, None]
    return rows, gelu(rows @ up.t() + d["bias"].double()), u @ down.t() + h, u.abs() @ down.abs().t() + h.abs(), rows.abs() @ up.abs().t()


@pytest.mark.parametrize("m,token", [(1, True), (6, True), (16, True), (1, False), (40, False), (300, False)])
def test_feed_forward_block(cuda_device, m, token):
    hid, f = 320, 1024
    d = mlp_weights(hid, f)
    x, res = randn(m, hid, seed=1).to(F16), randn(m, hid, seed=2).to(F16)
    before = res.clone()
    block = Mlp(d, m, hid, f)
    y = (block.token if token else block.prompt)(x, res)
    _, want = norm_of(x, before, d["norm"], 1e-6)
    assert_rows8(block.h8, block.hs, want)
    rows, u, out, mag, mag_u = mlp_plain(d, x, before, token, block)
    assert_fp16_close(block.u, u, mag_u * (80 * 2.0 ** -22) + (u.abs() + 8) * 2.0 ** -20)
    # the residual enters rounded to fp16 (2^-11 of it)
    assert_fp16_close(y, out, mag * (80 * 2.0 ** -22) + (x.double() + before.double()).abs() * 2.0 ** -11)


@pytest.mark.parametrize("m,token", [(1, True), (4, False), (200, False)])
def test_captured_and_replayed_and_on_another_stream(cuda_device, m, token):
    hid, f = 320, 1024
    d = mlp_weights(hid, f)
    x0, res0 = randn(m, hid, seed=1).to(F16), randn(m, hid, seed=2).to(F16)
    x1, res1 = randn(m, hid, seed=3).to(F16), randn(m, hid, seed=4).to(F16)
    block = Mlp(d, m, hid, f)
    run = block.token if token else block.prompt
    want = [run(a.clone(), b.clone()).clone() for a, b in ((x0, res0), (x1, res1))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = Mlp(d, m, hid, f)
        got = (other.token if token else other.prompt)(x0.clone(), res0.clone()).clone()
    side.synchronize()
    assert torch.equal(got, want[0])
    x, res = x0.clone(), res0.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run(x, res)
    for a, b, w in ((x0, res0, want[0]), (x1, res1, want[1]), (x0, res0, want[0])):
        x.copy_(a)
        res.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, w)
    ops.poll_status()
