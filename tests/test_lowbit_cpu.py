"""The low-bit path without a GPU: what its entry points refuse, before any device is touched, and the 4-bit form of
weights."""
import ctypes

import pytest
import torch

from dtas_b200 import _abi, ops, weights
from dtas_b200.build import build_library


@pytest.fixture(scope="module")
def lib():
    build_library()
    return _abi.lib()


@pytest.fixture(scope="module")
def p():
    buf = (ctypes.c_char * 64)()
    yield ctypes.addressof(buf)


def test_add_rms_norm_refuses(lib, p):
    call = lib.dtas_add_rms_norm
    ok = dict(x=p, res=p, w=p, y=p, ro=None, s=p, m=1, n=8, i=_abi.F16, o=_abi.E4M3)

    def rc(**kw):
        a = {**ok, **kw}
        return call(a["x"], a["res"], a["w"], a["y"], a["ro"], a["s"], a["m"], a["n"], 1e-6, a["i"], a["o"], 0, None)

    for bad in (dict(x=None), dict(w=None), dict(y=None), dict(s=None), dict(m=0), dict(m=-1), dict(n=0), dict(n=1 << 31)):
        assert rc(**bad) == _abi.EINVAL, bad
    assert rc(i=_abi.I8) == rc(i=9) == rc(o=_abi.F32) == rc(o=9) == _abi.EUNSUPPORTED
    assert b"add_rms_norm" in lib.dtas_last_error()


def test_quantize_refuses(lib, p):
    call = lib.dtas_quantize
    for bad in ((None, p, p, 1, 8), (p, None, p, 1, 8), (p, p, None, 1, 8), (p, p, p, 0, 8), (p, p, p, 1, 0)):
        assert call(*bad, _abi.F16, _abi.I8, 0, None) == _abi.EINVAL
    assert call(p, p, p, 1, 8, _abi.F16, _abi.F16, 0, None) == _abi.EUNSUPPORTED
    assert call(p, p, p, 1, 8, _abi.E4M3, _abi.I8, 0, None) == _abi.EUNSUPPORTED


def test_gemv_w4_refuses(lib, p):
    ok = dict(x=p, xs=None, w=p, ws=p, z=None, b=None, r1=None, r2=None, y=p, m=1, n=16, k=64, g=32, act=0, xd=_abi.F16, od=_abi.F16)

    def rc(**kw):
        a = {**ok, **kw}
        return lib.dtas_gemv_w4(*[a[x] for x in ("x", "xs", "w", "ws", "z", "b", "r1", "r2", "y", "m", "n", "k", "g", "act", "xd", "od")], 0, None)

    for bad in (dict(x=None), dict(w=None), dict(ws=None), dict(y=None), dict(m=0), dict(n=0), dict(k=0), dict(k=63, g=63), dict(g=0),
                dict(g=48), dict(g=-32), dict(act=7), dict(r2=p), dict(xs=p), dict(xd=_abi.I8), dict(xd=_abi.E4M3), dict(n=1 << 31),
                dict(k=1 << 31, g=32)):
        assert rc(**bad) == _abi.EINVAL, bad
    for bad in (dict(m=17), dict(xd=_abi.F32), dict(od=_abi.I8)):
        assert rc(**bad) == _abi.EUNSUPPORTED, bad


def test_gemm_f8_refuses(lib, p):
    ok = dict(x=p, w=p, xs=p, ws=p, b=None, r1=None, r2=None, y=p, m=1, n=16, k=64, ldy=16, ldr=0, act=0, od=_abi.F16)

    def rc(**kw):
        a = {**ok, **kw}
        return lib.dtas_gemm_nt_f8(*[a[x] for x in ("x", "w", "xs", "ws", "b", "r1", "r2", "y", "m", "n", "k", "ldy", "ldr", "act", "od")], 0, None)

    for bad in (dict(x=None), dict(w=None), dict(xs=None), dict(ws=None), dict(y=None), dict(m=0), dict(n=0), dict(k=-1), dict(ldy=15),
                dict(r1=p, ldr=8), dict(r2=p), dict(act=3)):
        assert rc(**bad) == _abi.EINVAL, bad
    assert rc(od=_abi.E4M3) == _abi.EUNSUPPORTED


def test_ops_refuse_cpu_tensors():
    x, w = torch.zeros(2, 64, dtype=torch.float16), torch.ones(64, dtype=torch.float16)
    q, s = torch.empty(2, 64, dtype=torch.int8), torch.empty(2)
    x8 = torch.zeros(2, 64).to(torch.float8_e4m3fn)
    for call in (lambda: ops.add_rms_norm(x, x, w, q, scale=s), lambda: ops.quantize(x, q, s),
                 lambda: ops.gemv_w4(x, torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 1, dtype=torch.float16), x[:, :8].contiguous()),
                 lambda: ops.gemm_nt_f8(x8, x8, s, s, torch.empty(2, 2, dtype=torch.float16))):
        with pytest.raises(_abi.DtasError) as e:
            call()
        assert e.value.code == _abi.EINVAL


def test_variants_have_names(lib):
    assert _abi.variant_of("add_rms_norm", 1, 4096) == "add_rms_norm_vec8_tpr512_ch1"
    assert _abi.variant_of("quantize", 8192, 11008) == "quantize_vec8_tpr352_ch4"
    assert _abi.variant_of("add_rms_norm", 8192, 4096) == "add_rms_norm_vec8_tpr128_ch4_stream"
    assert _abi.variant_of("add_rms_norm", 600, 1024) == "add_rms_norm_vec8_tpr128_ch1"
    assert _abi.variant_of("quantize", 8192, 1024) == "quantize_vec8_tpr64_ch2_stream"
    assert _abi.variant_of("add_rms_norm", 4, 16383) == "add_rms_norm_vec8_edge_tpr544_ch4_stream"
    assert _abi.variant_of("quantize", 1, 101) == "quantize_vec8_edge_tpr32_ch1"
    assert _abi.variant_of("add_rms_norm", 2, 1 << 20).startswith("add_rms_norm_long")
    assert "mma_m8" in _abi.variant_of("gemv_w4", 1, 4096, 4096) and "scalar" in _abi.variant_of("gemv_w4", 1, 4096, 34)
    assert _abi.variant_of("gemm_f8", 8192, 22016, 4096) == "f8_" + _abi.variant_of("gemm", 8192, 22016, 2048)
    assert _abi.variant_of("gemm_f8", 4, 64, 24) == "gemm_f8_simt_fallback"


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("n,k,group", [(3, 64, 32), (5, 256, 128), (2, 30, 15)])
def test_w4_form_of_weights(n, k, group, zero_points):
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(k)) * 0.1 + 0.02
    w[0, :group] = 0
    codes, scale, zero = weights.quantize_w4(w, group, zero_points)
    assert codes.dtype == torch.uint8 and codes.shape == (n, k // 2) and scale.shape == (n, k // group) and (zero is not None) == zero_points
    back = weights.dequantize_w4(codes, scale, zero, dtype=torch.float32)
    # half a step of the group; with zero points the zero is rounded too (another half), and the fp16 scale is off by 2^-11 of
    # itself, over at most 8 steps (15 with zero points) to the end of the range
    steps = (0.5 + 0.5 + 15 * 2 ** -11) if zero_points else (0.5 + 8 * 2 ** -11)
    tol = scale.float().repeat_interleave(group, 1) * steps + 1e-7
    assert ((back - w).abs() <= tol).all()
    assert (back[0, :group] == 0).all()
    with pytest.raises(_abi.DtasError):
        weights.quantize_w4(w, 7)
