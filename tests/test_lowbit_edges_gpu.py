"""The low-bit path on the GPU where a result is known exactly, and at its edges: values halfway between two 8-bit ones, products of
small whole numbers, residuals of other shapes and strides, infinities, odd addresses, stream order.

The products' operands are whole numbers and powers of two wherever a result is compared for equality: every partial sum is then a
whole number below 2^24 (times a power of two) and exact in fp32 whatever its order, so the one rounding to fp16 is all there
is, and a k that is lost, taken twice or scaled by another group's scale shows."""
import math

import pytest
import torch

from dtas_b200 import _abi, ops, weights

from tests.test_lowbit_gpu import CODES, SMALL_CODES, assert_fp16_close, gelu, randn

pytestmark = pytest.mark.gpu

F16, F32, I8, E4M3 = torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn
Q = {I8: 127.0, E4M3: 448.0}


# ---- values halfway between two 8-bit ones -----------------------------------------------------------
def halfway(dtype):
    """Every number halfway between neighbours of dtype, both signs, fp64."""
    if dtype == I8:
        t = torch.arange(0, 127, dtype=torch.float64) + 0.5
    else:
        steps = [torch.arange(0, 8, dtype=torch.float64) * 2.0 ** -9 + 2.0 ** -10]
        steps += [(torch.arange(8, 16, dtype=torch.float64) + 0.5) * 2.0 ** (e - 3) for e in range(-6, 9)]
        t = torch.cat(steps)
        t = t[t < 448]
    return torch.cat((t, -t))


def rows_of_halves(dtype, in_dtype, width):
    """Rows v with a maximum top such that v Q / top is halfway between two 8-bit values, all of it exact: with an odd s,
    v = t s / unit and top = Q s / unit for the halfway numbers t.  -> v, the t, both fp64 [rows, width]"""
    t = halfway(dtype)
    unit = 64.0 if dtype == E4M3 else 1.0
    if in_dtype == F16:        # s times the bits of t, 5 or 8 of them, within the 11 of fp16
        factors = range(1, 64, 2) if dtype == E4M3 else range(1, 8, 2)
        factors = [float(s) for s in factors]
    else:                      # 24 bits, over the range of fp32 exponents as well
        factors = [float(2 * s + 1) * 2.0 ** e for s, e in zip(range(0, 30000, 311), [0, -3, 20, -60, 70, -100, 95, -115, 0, 0] * 10)]
    v = torch.zeros(len(factors), width, dtype=torch.float64)
    want = torch.zeros_like(v)
    for i, s in enumerate(factors):
        v[i, 0], want[i, 0] = Q[dtype] * s / unit, Q[dtype]
        v[i, 1:1 + len(t)], want[i, 1:1 + len(t)] = t * s / unit, t
    assert torch.equal(v.to(in_dtype).double(), v)
    return v, want


def to_even(t, dtype):
    return t.round().to(I8) if dtype == I8 else t.to(F32).to(E4M3)      # t is an fp32 number: one rounding, to even


@pytest.mark.parametrize("width", [264, 271, 40001])
@pytest.mark.parametrize("in_dtype", [F16, F32])
@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_halves_go_to_the_even_value(cuda_device, dtype, in_dtype, width):
    v, t = rows_of_halves(dtype, in_dtype, width)
    m, want = len(v), to_even(t, dtype).cuda()
    buf = torch.zeros(m * width + 8, dtype=in_dtype, device="cuda")
    for off in (0, 1):                                                       # 16-byte vectors, and one element at a time
        x = buf[off:off + m * width].view(m, width)
        x.copy_(v)
        q, scale = torch.empty(m, width, dtype=dtype, device="cuda"), torch.empty(m, device="cuda")
        ops.quantize(x, q, scale)
        assert torch.equal(q.float(), want.float())
        top = v.abs().amax(-1).cuda()
        assert ((scale.double() - top / Q[dtype]).abs() <= top / Q[dtype] * 2.0 ** -24 + 2.0 ** -150).all()
        # through the norm, weights of one: its factor cancels, and the sum of two halves of v is v
        weight = torch.ones(width, dtype=F16, device="cuda")
        sane = (top < 1e18) & (top > 1e-15)                                  # squares within fp32
        ops.add_rms_norm(x, None, weight, q, scale=scale)
        assert torch.equal(q.float()[sane], want.float()[sane])
        if in_dtype == F32:
            half = x / 2
            ops.add_rms_norm(half, half, weight, q, scale=scale)
            assert torch.equal(q.float()[sane], want.float()[sane])


@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_rows_of_fp16_numbers_are_rounded_once(cuda_device, dtype):
    """Of fp16 rows the exact quotient is known: v Q is a number of at most 18 bits, and a quotient that is not halfway
    is further from there than 2^-19 of itself."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.randn(300, 4096, generator=g, device="cuda") * 8).to(F16)
    q, scale = torch.empty(300, 4096, dtype=dtype, device="cuda"), torch.empty(300, device="cuda")
    ops.quantize(x, q, scale)
    y = x.double() * Q[dtype] / x.double().abs().amax(-1, keepdim=True)
    assert torch.equal(q.float(), (y.round() if dtype == I8 else y.to(F32).to(E4M3)).float())


@pytest.mark.parametrize("h", [600, 1030, 4100, 8000, 8720, 17408, 20000])
def test_rows_at_odd_addresses_are_the_same_rows(cuda_device, h):
    """Neither a maximum nor a product depends on how a row is cut: the 8-bit rows are those of the aligned call."""
    m = 5
    for in_dtype in (F16, F32):
        x, res, weight = randn(m, h, seed=1).to(in_dtype), randn(m, h, seed=2).to(in_dtype), (1 + randn(h, seed=3, scale=0.1)).to(F16)
        buf = torch.zeros(m * h + 8, dtype=in_dtype, device="cuda")
        odd = buf[3:3 + m * h].view(m, h)
        odd.copy_(x)
        for dtype in (I8, E4M3):
            rows, scales, sums = [], [], []
            for a in (x, odd):
                out = torch.zeros(m * h + 8, dtype=torch.uint8, device="cuda")
                q = out[a is odd:][:m * h].view(dtype).view(m, h)
                scale, total = torch.empty(m, device="cuda"), torch.empty_like(x)
                ops.quantize(a, q, scale)
                rows.append(q.float()), scales.append(scale)
                q, s = torch.empty(m, h, dtype=dtype, device="cuda"), torch.empty(m, device="cuda")
                ops.add_rms_norm(a, res, weight, q, res_out=total, scale=s)
                rows.append(q.float()), scales.append(s), sums.append(total)
                assert (out[m * h + (a is odd):] == 0).all()
            assert torch.equal(rows[0], rows[2]) and torch.equal(rows[1], rows[3]) and torch.equal(sums[0], sums[1])
            assert torch.equal(scales[0], scales[2])
            assert ((scales[1] - scales[3]).abs() <= scales[1] * 2.0 ** -18).all()      # another order of the sum of squares


# ---- products of whole numbers -----------------------------------------------------------------------
def whole(*shape, top, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-top, top + 1, shape, generator=g, device="cuda")


def power(*shape, lo, hi, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return 2.0 ** torch.randint(lo, hi + 1, shape, generator=g, device="cuda").double()


W4_SHAPES = [(1, 32, 32), (70, 32, 32), (33, 1056, 32), (40, 64, 64), (31, 192, 64), (100, 4096, 128), (64, 4064, 32), (4099, 256, 32), (50, 11008, 128),
             (300, 20480, 64), (40, 768, 384), (70, 1536, 512), (35, 640, 640), (260, 2560, 64), (17, 60, 30), (9, 6, 3), (12, 2, 1)]


@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("x_dtype", [F16, I8, E4M3])
@pytest.mark.parametrize("n,k,group", W4_SHAPES)
def test_gemv_w4_of_whole_numbers(cuda_device, n, k, group, x_dtype, zero):
    for m in (1, 3, 8, 9, 16):
        x = whole(m, k, top=2, seed=m)
        codes = whole(n, k, top=7, seed=k) + 7 + (whole(n, k, top=1, seed=k + 1) > 0)       # 0 .. 15
        scales = power(n, k // group, lo=-2, hi=1, seed=n)
        zeros = (whole(n, k // group, top=7, seed=5) + 8).to(torch.uint8) if zero else None   # 1 .. 15
        x_scale = None if x_dtype == F16 else power(m, lo=-3, hi=3, seed=6).float()
        w = w4_matrix(codes, scales, zeros)
        want = (x.double() @ w.t()) * (1.0 if x_scale is None else x_scale.double()[:, None])
        bias, r1, r2 = (whole(*s, top=64, seed=7).to(F16) for s in ((n,), (m, n), (m, n)))
        # a row's sums: at most 2 * 15 * 20480 times a scale of 2, in steps of 2^-2, so below 2^23 steps; the row's scale moves
        # the exponent alone, and bias and residuals, up to 192 in steps of 1, add less than 2^13 steps of 2^-5
        for kw, add in (({}, 0), ({"bias": bias}, bias.double()), ({"res1": r1, "res2": r2}, r1.double() + r2.double())):
            out = torch.empty(m, n, dtype=F16, device="cuda")
            ops.gemv_w4(x.to(x_dtype if x_dtype != E4M3 else F32).to(x_dtype), weights.pack_w4(codes.to(torch.uint8)), scales.to(F16), out,
                        w_zero=zeros, x_scale=x_scale, **kw)
            assert torch.equal(out.float(), (want + add).to(F32).to(F16).float()), (m, list(kw))


@pytest.mark.parametrize("x_dtype", [F16, I8])
@pytest.mark.parametrize("m,n,k,group", [(1, 300, 4096, 128), (5, 300, 4096, 32), (16, 300, 11008, 128), (9, 200, 20480, 64), (2, 100, 4064, 32)])
def test_gemv_w4_roundings(cuda_device, m, n, k, group, x_dtype):
    """Accumulators of the MMAs restart with every group, or every 128 k of a longer one, so they see at most four steps, of two
    truncations to 2^-23 each, of sums bounded by the codes' (30 s |x|, as zero points enter apart); the sums of x
    a dozen roundings of 2^-24.  Two fused multiply-adds per group in a row's fp32 sum, and the joins of at most 12 warps and 8 CTAs,
    are roundings of 2^-24 of a sum bounded by |x| |w|."""
    _, codes, packed, scales, zeros = w4_operands(m, n, k, group, True, seed=k)
    x = randn(m, k, seed=m)
    x_scale = None
    if x_dtype == I8:
        x_scale, x = torch.full((m,), 0.03, device="cuda"), (x * 30).round().clamp(-127, 127)
    w = w4_matrix(codes, scales, zeros)
    out = torch.empty(m, n, dtype=F16, device="cuda")
    ops.gemv_w4(x.to(x_dtype), packed, scales, out, w_zero=zeros, x_scale=x_scale)
    xd = x.to(x_dtype).double() * (1.0 if x_scale is None else x_scale.double()[:, None])
    codes_mag = xd.abs() @ (30 * scales.double()).repeat_interleave(group, 1).t()
    sum_mag = xd.abs() @ w.abs().t()
    assert_fp16_close(out, xd @ w.t(), codes_mag * ((8 + 6) * 2.0 ** -23) + sum_mag * ((2 * k // min(group, 128) + 24) * 2.0 ** -24))


@pytest.fixture
def in_kernel():
    lib = _abi.lib()
    yield lambda code: _abi.check(lib.dtas_gemm_set_override(*code))
    lib.dtas_gemm_set_override(0, 0)


@pytest.mark.parametrize("n", [328, 333, 512])
@pytest.mark.parametrize("m,code", [(m, c) for m in (200, 333) for c in CODES] + [(m, c) for m in (1, 20, 50) for c in SMALL_CODES] + [(513, (0, 0)), (2, (0, 0))])
def test_gemm_f8_of_whole_numbers_in_every_kernel(cuda_device, in_kernel, m, code, n):
    """Residuals as views of wider buffers, one and two of them, ragged and whole tiles; results as they are, as fp32 and in a slab."""
    k = 1616
    x, w = whole(m, k, top=2, seed=m), whole(n, k, top=2, seed=n)
    sx, sw = power(m, lo=-3, hi=3, seed=1), power(n, lo=-3, hi=3, seed=2)
    y = (x.double() @ w.double().t()) * sx[:, None] * sw
    bias = whole(n, top=64, seed=3).to(F16)
    wide = whole(2, m, n + 24, top=64, seed=4).to(F16)
    r1, r2 = wide[0][:, 8:8 + n], wide[1][:, 16:16 + n]
    x8, w8 = x.float().to(E4M3), w.float().to(E4M3)
    in_kernel(code)
    for kw, add in (({}, 0), ({"bias": bias}, bias.double()), ({"res1": r1}, r1.double()), ({"bias": bias, "res1": r1, "res2": r2}, bias.double() + r1.double() + r2.double()),
                    ({"res1": r1.contiguous(), "res2": r2.contiguous()}, r1.double() + r2.double())):
        want = (y + add).to(F32).to(F16)
        for dtype in (F16, F32):
            buf = torch.full((m, n + 40), 3.0, dtype=dtype, device="cuda")
            for out in (buf[:, 16:16 + n], torch.empty(m, n, dtype=dtype, device="cuda")):
                ops.gemm_nt_f8(x8, w8, sx.float(), sw.float(), out, **kw)
                assert torch.equal(out.float(), want.float()), (list(kw), dtype)
            assert (buf[:, :16] == 3.0).all() and (buf[:, 16 + n:] == 3.0).all()
    ops.poll_status()


@pytest.mark.parametrize("n", [328, 512])
@pytest.mark.parametrize("m,code", [(333, c) for c in CODES] + [(20, c) for c in SMALL_CODES])
def test_gemm_f8_activation_and_two_residuals(cuda_device, in_kernel, m, code, n):
    """Sums as above are exact, so what is left is the activation (erf good to 5e-7, a few operations) and three additions."""
    k = 400
    x, w = whole(m, k, top=2, seed=m), whole(n, k, top=2, seed=n)
    sx, sw = power(m, lo=-6, hi=-3, seed=1), power(n, lo=-2, hi=0, seed=2)
    bias, r1, r2 = randn(n, seed=3).to(F16), randn(m, n, seed=4).to(F16), randn(m, n, seed=5).to(F16)
    t = (x.double() @ w.double().t()) * sx[:, None] * sw + bias.double()
    in_kernel(code)
    out = torch.empty(m, n, dtype=F16, device="cuda")
    ops.gemm_nt_f8(x.float().to(E4M3), w.float().to(E4M3), sx.float(), sw.float(), out, bias=bias, act="gelu", res1=r1, res2=r2)
    mag = t.abs() + r1.double().abs() + r2.double().abs()
    assert_fp16_close(out, gelu(t) + r1.double() + r2.double(), mag * 2.0 ** -20)
    ops.poll_status()


@pytest.mark.parametrize("m", [300, 2100])
def test_gemm_into_its_own_residual(cuda_device, m):
    n, k = 264, 128
    x, w, r, r2 = (whole(*s, top=2, seed=i).to(F16) for i, s in enumerate(((m, k), (n, k), (m, n), (m, n))))
    want = x.double() @ w.double().t() + r.double() + r2.double()
    for first in (True, False):
        out = r.clone()
        ops.gemm_nt(x, w, out, res1=out if first else r2, res2=r2 if first else out)
        assert torch.equal(out.double(), want)
        row, other = r[:1].clone(), r2[:1]
        ops.gemv(x[:1], w, row, res1=row if first else other, res2=other if first else row)
        assert torch.equal(row.double(), want[:1])


@pytest.mark.parametrize("n", [328, 333])
@pytest.mark.parametrize("m,code", [(m, c) for m in (200, 333) for c in CODES] + [(m, c) for m in (1, 20, 50) for c in SMALL_CODES] + [(2100, (0, 0))])
def test_low_bit_products_into_their_own_residual(cuda_device, in_kernel, m, code, n):
    """The residual stream as both an operand and the result: every element is read before it is stored."""
    k = 400
    x, w = whole(m, k, top=2, seed=m), whole(n, k, top=2, seed=n)
    r, r2 = whole(m, n, top=64, seed=4).to(F16), whole(m, n, top=64, seed=5).to(F16)
    one = torch.ones(max(m, n), device="cuda")
    in_kernel(code)
    want = x.double() @ w.double().t() + r.double() + r2.double()
    for first in (True, False):
        out = r.clone()
        ops.gemm_nt_f8(x.float().to(E4M3), w.float().to(E4M3), one[:m], one[:n], out, res1=out if first else r2, res2=r2 if first else out)
        assert torch.equal(out.double(), want)
    if m <= 16:
        codes = (w + 8).to(torch.uint8)
        out = r.clone()
        ops.gemv_w4(x.to(F16), weights.pack_w4(codes), torch.ones(n, 1, dtype=F16, device="cuda"), out, res1=out, res2=r2)
        assert torch.equal(out.double(), want)


# ---- residuals of other shapes and strides -----------------------------------------------------------
def test_residuals_of_other_shapes_are_refused(cuda_device):
    m, n, k = 12, 24, 64
    z = lambda *shape, dt=F16: torch.zeros(*shape, dtype=dt, device="cuda")  # noqa: E731
    x, w, x8, w8 = z(m, k), z(n, k), z(m, k, dt=F32).to(E4M3), z(n, k, dt=F32).to(E4M3)
    codes, scales = z(n, k // 2, dt=torch.uint8), z(n, 2)
    out = torch.full((m, n), 3.0, dtype=F16, device="cuda")
    for r in (z(n, m), z(n).expand(m, n), z(1, n).expand(m, n), z(2 * m, n // 2), z(m * n), z(m, n).float(), z(m - 1, n)):
        for kw in ({"res1": r}, {"res1": z(m, n), "res2": r}):
            for call in (lambda: ops.gemm_nt_f8(x8, w8, z(m, dt=F32), z(n, dt=F32), out, **kw), lambda: ops.gemv_w4(x, codes, scales, out, **kw),
                         lambda: ops.gemm_nt(x, w, out, **kw)):
                with pytest.raises(_abi.DtasError):
                    call()
    assert (out == 3.0).all()


def test_rows_without_a_scale_are_refused(cuda_device):
    x, q = torch.zeros(2, 8, dtype=F16, device="cuda"), torch.zeros(2, 8, dtype=I8, device="cuda")
    for call in (lambda: ops.quantize(x, q, None), lambda: ops.add_rms_norm(x, None, x[0], q)):
        with pytest.raises(_abi.DtasError) as e:
            call()
        assert e.value.code == _abi.EINVAL


# ---- 4-bit products: what is not finite --------------------------------------------------------------
def w4_operands(m, n, k, group, zero, seed=0):
    """x, codes [N, K], packed codes, scales, zero points or None."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.01 + 0.01 * torch.rand(n, k // group, generator=g, device="cuda")).to(F16)
    zeros = torch.randint(0, 16, (n, k // group), generator=g, device="cuda", dtype=torch.uint8) if zero else None
    return torch.randn(m, k, generator=g, device="cuda").to(F16), codes, weights.pack_w4(codes), scales, zeros


def w4_matrix(codes, scales, zeros):
    n, groups = scales.shape
    z = 8.0 if zeros is None else zeros.double()[..., None]
    return ((codes.double().view(n, groups, -1) - z) * scales.double()[..., None]).view(n, -1)


@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("m,n,k,group", [(4, 70, 128, 64), (4, 70, 60, 30), (1, 33, 4096, 128), (7, 100, 1056, 32), (16, 200, 11008, 128)])
def test_gemv_w4_infinities_are_those_of_the_formula(cuda_device, m, n, k, group, zero):
    """An infinite x gives an infinity by the sign of code - zero, a NaN where that is 0; two of them, or a NaN, what their sum is.
    The same from both kernels, and nothing in the other rows."""
    x, codes, packed, scales, zeros = w4_operands(m, n, k, group, zero, seed=k)
    x[0, k // 3] = math.inf
    if m > 2:
        x[1, k - 1], x[1, 2] = -math.inf, math.inf
        x[2, 5] = math.nan
    scales[5, 0] = math.inf
    w = w4_matrix(codes, scales, zeros)
    out = torch.empty(m, n, dtype=F16, device="cuda")
    ops.gemv_w4(x, packed, scales, out, w_zero=zeros)
    # the products one by one: a matrix product may take infinities in any order, but no order changes these
    for i in range(m):
        want = (x[i].double() * w).sum(-1)
        assert torch.equal(torch.isnan(out[i]), torch.isnan(want)), i
        assert torch.equal(torch.isinf(out[i]), torch.isinf(want)), i
        inf = torch.isinf(want)
        assert torch.equal(out[i][inf].double(), want[inf])
        if i not in (0, 1, 2):
            assert torch.isfinite(out[i][torch.arange(n, device="cuda") != 5].float()).all()


@pytest.mark.parametrize("k", [128, 60])
def test_gemv_w4_with_row_scales_at_the_ends_of_fp32(cuda_device, k):
    """Rows of 8 bits whose scale is very large or very small, as those of fp32 rows may be: their sums times the scale, 0 where the sum
    is 0."""
    n, group = 40, k // 2
    _, codes, packed, _, _ = w4_operands(1, n, k, group, False, seed=1)
    codes[7] = 8                                           # a row of zeros: its sums are 0 whatever the scale
    packed = weights.pack_w4(codes)
    scales = torch.full((n, 2), 2.0 ** -14, dtype=F16, device="cuda")
    x = torch.ones(4, k, dtype=I8, device="cuda")
    x_scale = torch.tensor([2.0 ** 127, 2.0 ** 104, 2.0 ** -140, 1.0], device="cuda")
    out = torch.empty(4, n, dtype=F32, device="cuda")
    ops.gemv_w4(x, packed, scales, out, x_scale=x_scale)
    want = ((codes.double() - 8).sum(-1) * 2.0 ** -14 * x_scale.double()[:, None]).to(F16).float()
    assert torch.equal(out, want)


# ---- stream order ------------------------------------------------------------------------------------
class Chain:
    """Every operand of a low-bit call - activations, scales, weights, biases - is written by the call right before
    it, buffers are reused, and nothing synchronises in between: kernels start while the one before them still runs."""

    def __init__(self, m, h, f):
        g = torch.Generator(device="cuda").manual_seed(5)
        rand = lambda *shape, s=1.0: (torch.randn(*shape, generator=g, device="cuda") * s).to(F16)  # noqa: E731
        new = lambda *shape, dt=F16: torch.zeros(*shape, dtype=dt, device="cuda")  # noqa: E731
        self.m = m
        self.norms, self.biases = [rand(1, h) for _ in range(2)], [rand(1, f, s=0.1) for _ in range(2)]
        self.downs = [rand(h, f, s=0.05) for _ in range(2)]
        self.ups = [weights.quantize_w4(rand(f, h, s=0.05), 32, True) for _ in range(2)]
        self.x0, self.res0 = rand(m, h), rand(m, h)
        self.x, self.res, self.norm, self.bias = new(m, h), new(m, h), new(1, h), new(1, f)
        self.codes, self.scales, self.zeros = (torch.zeros_like(t) for t in self.ups[0])
        self.h8, self.hs, self.u = new(m, h, dt=E4M3), new(m, dt=F32), new(m, f)
        self.u8, self.us, self.w8, self.ws, self.y = new(m, f, dt=E4M3), new(m, dt=F32), new(h, f, dt=E4M3), new(h, dt=F32), new(m, h)
        self.outs = [new(m, h) for _ in range(4)]

    def run(self, sync):
        def call(op, *args, **kw):
            op(*args, **kw)
            if sync:
                torch.cuda.synchronize()

        call(ops.copy, self.x0, self.x)
        call(ops.copy, self.res0, self.res)
        for i in range(4):
            up = self.ups[i % 2]
            call(ops.copy, self.norms[i % 2], self.norm)
            call(ops.add_rms_norm, self.x, self.res, self.norm, self.h8, res_out=self.res, scale=self.hs)
            call(ops.copy, up[2].view(I8), self.zeros.view(I8))
            call(ops.copy, up[1], self.scales)
            call(ops.copy, up[0].view(I8), self.codes.view(I8))
            call(ops.copy, self.biases[i % 2], self.bias)
            call(ops.gemv_w4, self.h8, self.codes, self.scales, self.u, w_zero=self.zeros, x_scale=self.hs, bias=self.bias, act="gelu")
            call(ops.gemv_w4, self.res, self.codes, self.scales, self.u, w_zero=self.zeros, res1=self.u)
            call(ops.quantize, self.downs[i % 2], self.w8, self.ws)
            call(ops.quantize, self.u, self.u8, self.us)
            call(ops.gemm_nt_f8, self.u8, self.w8, self.us, self.ws, self.y, res1=self.res)
            call(ops.add_rms_norm, self.y, None, self.norm, self.x)
            call(ops.copy, self.x, self.outs[i])
        return [o.clone() for o in self.outs]


@pytest.mark.parametrize("m,h,f", [(1, 1024, 4096), (16, 2560, 2816), (5, 1025 * 32, 96), (3, 4096, 11008)])
def test_calls_keep_stream_order(cuda_device, m, h, f):
    chain = Chain(m, h, f)
    want = chain.run(sync=True)
    assert all(torch.isfinite(o.float()).all() for o in want) and not torch.equal(want[0], want[1])
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(chain.run(sync=False), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain.run(sync=False)
    for _ in range(20):
        for o in chain.outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(chain.outs, want))
    ops.poll_status()


# ---- the calls' other forms: sizes, shapes, threads ----------------------------------------------------
@pytest.mark.parametrize("h", [16384, 16383])
def test_rows_beyond_32_bit_offsets(cuda_device, h):
    """More than 2^31 elements: rows on both sides of the border are those that a call of their own gives."""
    m = 2 ** 31 // h + 40
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(m, h, dtype=F16, device="cuda").normal_(generator=g)
    weight = (1 + randn(h, seed=3, scale=0.1)).to(F16)
    rows = torch.tensor([0, 1, m // 2, m - 41, m - 40, m - 39, m - 2, m - 1], device="cuda")
    some = x[rows].clone()
    q, scale = torch.empty(m, h, dtype=I8, device="cuda"), torch.empty(m, device="cuda")
    q1, s1 = torch.empty(len(rows), h, dtype=I8, device="cuda"), torch.empty(len(rows), device="cuda")
    ops.quantize(x, q, scale)
    ops.quantize(some, q1, s1)
    assert torch.equal(q[rows], q1) and torch.equal(scale[rows], s1)
    twice = some.float() * 2
    ops.add_rms_norm(some, some, weight, q1, scale=s1)
    ops.add_rms_norm(x, x, weight, q, res_out=x, scale=scale)
    assert torch.equal(q[rows], q1) and ((scale[rows] - s1).abs() <= s1 * 2.0 ** -18).all()
    assert torch.equal(x[rows].float(), twice)


def test_products_beyond_32_bit_offsets(cuda_device):
    """Weights, results and residuals of more than 2^31 elements."""
    def eight(t):
        return t.float().to(E4M3)

    m, n, k = 270000, 8192, 64                                    # y and the residual, which is y
    x, w = whole(m, k, top=2, seed=1), whole(n, k, top=2, seed=2)
    y = torch.ones(m, n, dtype=F16, device="cuda")
    ops.gemm_nt_f8(eight(x), eight(w), torch.ones(m, device="cuda"), torch.ones(n, device="cuda"), y, res1=y)
    rows = torch.tensor([0, 2 ** 31 // n - 1, 2 ** 31 // n, m - 1], device="cuda")
    assert torch.equal(y[rows].double(), x[rows].double() @ w.double().t() + 1)
    del y
    m, n, k = 3, 262145, 8208                                     # w, for both products
    x, w = whole(m, k, top=2, seed=1), torch.zeros(n, k, dtype=torch.uint8, device="cuda")
    rows = torch.tensor([0, 2 ** 31 // k, 2 ** 31 // k + 1, n - 1], device="cuda")
    w[rows] = (whole(4, k, top=7, seed=3) + 8).to(torch.uint8)
    y = torch.empty(m, n, dtype=F16, device="cuda")
    ops.gemm_nt_f8(eight(x), w.to(E4M3), torch.ones(m, device="cuda"), torch.ones(n, device="cuda"), y)
    assert torch.equal(y[:, rows].float(), (x.double() @ w[rows].double().t()).float().to(F16).float())
    m, n, k, group = 9, 1048577, 4096, 32                         # codes, and 2^27 scales
    x = whole(m, k, top=2, seed=1)
    codes = torch.full((n, k // 2), 0x88, dtype=torch.uint8, device="cuda")
    rows = torch.tensor([0, 2 ** 20 - 1, 2 ** 20, n - 1], device="cuda")
    some = whole(4, k, top=7, seed=3) + 8
    codes[rows] = weights.pack_w4(some.to(torch.uint8))
    y = torch.empty(m, n, dtype=F16, device="cuda")
    ops.gemv_w4(x.to(F16), codes, torch.ones(n, k // group, dtype=F16, device="cuda"), y)
    held = torch.stack((codes[rows] & 15, codes[rows] >> 4), -1).view(4, k).double() - 8      # the last two rows are one
    assert torch.equal(y[:, rows].float(), (x.double() @ held.t()).float().to(F16).float())
    y[:, rows] = 0
    assert (y == 0).all()
    ops.poll_status()


def test_operands_with_a_leading_unit_dimension(cuda_device):
    """[1, m, H] beside [m, H], in every operand that has rows."""
    m, n, k = 5, 48, 64
    lead = lambda t: t.unsqueeze(0)  # noqa: E731
    x, res, weight = randn(m, k, seed=1).to(F16), randn(m, k, seed=2).to(F16), (1 + randn(k, seed=3, scale=0.1)).to(F16)
    got = [[torch.empty(m, k, dtype=E4M3, device="cuda"), torch.empty(m, device="cuda"), torch.empty_like(x)] for _ in range(2)]
    ops.add_rms_norm(x, res, weight, got[0][0], res_out=got[0][2], scale=got[0][1])
    ops.add_rms_norm(lead(x), res, lead(lead(weight)), lead(got[1][0]), res_out=lead(got[1][2]), scale=lead(got[1][1]))
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(*got))
    rows, scale, _ = got[0]
    q, s = torch.empty_like(rows), torch.empty_like(scale)
    ops.quantize(lead(x), lead(q), s)
    ops.quantize(x, rows, scale)
    assert torch.equal(q.float(), rows.float()) and torch.equal(s, scale)
    r, bias = randn(m, n, seed=4).to(F16), randn(n, seed=5).to(F16)
    w8, ws = torch.empty(n, k, dtype=E4M3, device="cuda"), torch.empty(n, device="cuda")
    ops.quantize(randn(n, k, seed=6).to(F16), w8, ws)
    codes, scales, zeros = weights.quantize_w4(randn(n, k, seed=7), 32, True)
    wide = torch.zeros(1, m, 3 * n, dtype=F16, device="cuda")
    for call in (lambda a, b, o: ops.gemm_nt_f8(a, w8, scale, ws, o, bias=bias, res1=b, act="gelu"),
                 lambda a, b, o: ops.gemv_w4(a, codes, scales, o, w_zero=zeros, x_scale=scale, bias=bias, res1=b, act="gelu")):
        want = call(rows, r, torch.empty(m, n, dtype=F16, device="cuda"))
        assert torch.equal(call(lead(rows), lead(r), torch.empty(1, m, n, dtype=F16, device="cuda"))[0], want)
        assert torch.equal(call(lead(rows), r, torch.empty(m, n, dtype=F16, device="cuda")), want)
    slab = wide[:, :, n:2 * n]
    ops.gemm_nt_f8(lead(rows), w8, scale, ws, slab, bias=bias, res1=lead(r), act="gelu")
    assert torch.equal(slab[0], ops.gemm_nt_f8(rows, w8, scale, ws, torch.empty(m, n, dtype=F16, device="cuda"), bias=bias, res1=r, act="gelu"))
    assert (wide[:, :, :n] == 0).all() and (wide[:, :, 2 * n:] == 0).all()


def test_calls_from_several_threads(cuda_device):
    """Host threads with streams of their own, all calls at once: every one gets what it gets alone."""
    import threading
    chains = [Chain(m, 1024, 4096) for m in (1, 3, 8, 16)]
    want = [c.run(sync=True) for c in chains]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                got = chains[i].run(sync=False)
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    failed.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(chains))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    ops.poll_status()
