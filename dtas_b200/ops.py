"""Torch-tensor front end of the C ABI: one function per operator.

Calling convention follows the reference's packed functions: inputs first, the
pre-allocated output last (experiment/dtas_tuned/elementwise/cast/profile_cast.py:15-18);
the symbolic dim is read from the tensor shape, never passed
(experiment/dtas_tuned/elementwise/cast/top10_256/host.cc:52-53).  Tensors may be
`[m, H]` or the reference's `[1, m, H]`.  Every function launches on the current torch
stream of the tensor's device and returns the output tensor.
"""
import torch

from . import _abi

_L = None


def _lib():
    global _L
    if _L is None:
        _L = _abi.lib()
    return _L

_DTYPE_CODE = {torch.float16: _abi.F16, torch.float32: _abi.F32, torch.int8: _abi.I8}


def _chk(status):
    if status:
        _abi.check(status)


def _code(t):
    try:
        return _DTYPE_CODE[t.dtype]
    except KeyError:
        raise _abi.DtasError(_abi.EUNSUPPORTED, f"dtype {t.dtype} has no kernel") from None


def _rows_cols(t, name):
    """[m, H] or [1, m, H] -> (m, H)."""
    if t.dim() == 3 and t.shape[0] == 1:
        return int(t.shape[1]), int(t.shape[2])
    if t.dim() == 2:
        return int(t.shape[0]), int(t.shape[1])
    raise _abi.DtasError(_abi.EINVAL, f"{name}: expected [m, H] or [1, m, H], got {tuple(t.shape)}")


try:   # raw handle of the current stream without building a torch.cuda.Stream object
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:   # older / stripped builds
    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream


def _check(name, *tensors):
    """Device index and current raw stream; rejects CPU, mixed-device and strided tensors."""
    first = tensors[0]
    if not first.is_cuda:
        raise _abi.DtasError(_abi.EINVAL, f"{name}: tensors must live on a CUDA device, got {first.device}")
    dev = first.device
    for t in tensors:
        if not t.is_contiguous():
            raise _abi.DtasError(_abi.EINVAL, f"{name}: tensors must be contiguous")
        if t.device != dev:
            raise _abi.DtasError(_abi.EINVAL, f"{name}: tensors on different devices")
    index = dev.index
    return index, _raw_stream(index)


def _same_shape(name, a, b):
    if _rows_cols(a, name) != _rows_cols(b, name):
        raise _abi.DtasError(_abi.EINVAL, f"{name}: shape mismatch {tuple(a.shape)} vs {tuple(b.shape)}")


def cast(a, out):
    """out = a converted to out.dtype (fp32 -> fp16 round-to-nearest-even, or fp16 -> fp32)."""
    dev, st = _check("cast", a, out)
    _same_shape("cast", a, out)
    m, h = _rows_cols(a, "cast")
    _chk(_lib().dtas_cast(a.data_ptr(), out.data_ptr(), m, h, _code(a), _code(out), dev, st))
    return out


def add(a, b, out):
    """out = a + b, all three of one dtype (fp16, fp32 or int8)."""
    dev, st = _check("add", a, b, out)
    _same_shape("add", a, b)
    _same_shape("add", a, out)
    if not (a.dtype == b.dtype == out.dtype):
        raise _abi.DtasError(_abi.EINVAL, "add: dtypes differ")
    m, h = _rows_cols(a, "add")
    _chk(_lib().dtas_add(a.data_ptr(), b.data_ptr(), out.data_ptr(), m, h, _code(a), dev, st))
    return out


def copy(a, out):
    """out = a."""
    dev, st = _check("copy", a, out)
    _same_shape("copy", a, out)
    if a.dtype != out.dtype:
        raise _abi.DtasError(_abi.EINVAL, "copy: dtypes differ")
    m, h = _rows_cols(a, "copy")
    _chk(_lib().dtas_copy(a.data_ptr(), out.data_ptr(), m, h, _code(a), dev, st))
    return out


def peer_push(src, dsts):
    """Copies the contiguous tensor `src` to every tensor of `dsts`: views, on this device, of the
    same place in the other ranks' gather buffers (peer memory).  One launch, plain stores over
    NVLink, no cross-rank waiting: run a barrier across ranks before a gathered buffer is read."""
    import ctypes
    dev, st = _check("peer_push", src, *dsts)
    for d in dsts:
        if d.dtype != src.dtype or d.numel() != src.numel():
            raise _abi.DtasError(_abi.EINVAL, "peer_push: destination of another size or dtype")
    ptrs = (ctypes.c_void_p * len(dsts))(*[d.data_ptr() for d in dsts])
    _chk(_lib().dtas_peer_push(src.data_ptr(), ptrs, len(dsts), src.numel() * src.element_size(), dev, st))


def rms_norm(x, weight, out, eps=1e-6):
    """out = x * rsqrt(mean(x^2, -1) + eps) * weight; fp32 arithmetic, fp16 result."""
    dev, st = _check("rms_norm", x, weight, out)
    _same_shape("rms_norm", x, out)
    m, h = _rows_cols(x, "rms_norm")
    if weight.dtype != torch.float16 or weight.numel() != h or out.dtype != torch.float16:
        raise _abi.DtasError(_abi.EINVAL, "rms_norm: weight must be fp16 [H] and out fp16")
    _chk(_lib().dtas_rms_norm(x.data_ptr(), weight.data_ptr(), out.data_ptr(), m, h,
                                        float(eps), _code(x), dev, st))
    return out


def softmax(x, out):
    """out = softmax(x, dim=-1); fp32 arithmetic, fp16 result."""
    dev, st = _check("softmax", x, out)
    _same_shape("softmax", x, out)
    if out.dtype != torch.float16:
        raise _abi.DtasError(_abi.EINVAL, "softmax: out must be fp16")
    m, h = _rows_cols(x, "softmax")
    _chk(_lib().dtas_softmax(x.data_ptr(), out.data_ptr(), m, h, _code(x), dev, st))
    return out


def layer_norm(x, gamma, beta, out, eps=1e-5):
    """out = (x - mean) * rsqrt(var + eps) * gamma + beta; gamma/beta fp32 [H]; fp16 result."""
    dev, st = _check("layer_norm", x, gamma, beta, out)
    _same_shape("layer_norm", x, out)
    m, h = _rows_cols(x, "layer_norm")
    if gamma.dtype != torch.float32 or beta.dtype != torch.float32 or gamma.numel() != h or beta.numel() != h:
        raise _abi.DtasError(_abi.EINVAL, "layer_norm: gamma and beta must be fp32 [H]")
    if out.dtype != torch.float16:
        raise _abi.DtasError(_abi.EINVAL, "layer_norm: out must be fp16")
    _chk(_lib().dtas_layer_norm(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), out.data_ptr(),
                                          m, h, float(eps), _code(x), dev, st))
    return out


_ACTS = {None: _abi.ACT_NONE, "none": _abi.ACT_NONE, "gelu": _abi.ACT_GELU}


def _tail_args(name, out, n, rows, bias, res1, res2, act):
    """Checks the optional tail operands; -> (act code, out dtype code, ldr, fused?)."""
    if act not in _ACTS:
        raise _abi.DtasError(_abi.EINVAL, f"{name}: unknown activation {act!r} (None or 'gelu')")
    if out.dtype not in (torch.float16, torch.float32):
        raise _abi.DtasError(_abi.EUNSUPPORTED, f"{name}: the output must be fp16 or fp32, got {out.dtype}")
    if res1 is None and res2 is not None:
        raise _abi.DtasError(_abi.EINVAL, f"{name}: res2 without res1")
    if bias is not None and (bias.dtype != torch.float16 or bias.numel() != n or not bias.is_contiguous()):
        raise _abi.DtasError(_abi.EINVAL, f"{name}: bias must be a contiguous fp16 vector of N elements")
    ldr = 0
    for r in (res1, res2):
        if r is None:
            continue
        # rows of n elements, one behind the other, or [m, N] with rows further apart: nothing else may give the kernel a row
        # stride, for it would read rows where there are none (a row stride of 0, [N, m])
        shape = tuple(r.shape)
        if r.is_contiguous() and r.numel() == rows * n and (rows == 1 or shape[-1] == n):
            ld = n
        elif shape in ((rows, n), (1, rows, n)) and (n == 1 or r.stride(-1) == 1) and r.stride(-2) >= n:
            ld = int(r.stride(-2))
        else:
            ld = 0
        if r.dtype != torch.float16 or ld == 0:
            raise _abi.DtasError(_abi.EINVAL, f"{name}: residuals must be fp16 [m, N] with unit inner stride and rows that do not "
                                              f"overlap, got {r.dtype} {shape} with strides {tuple(r.stride())}")
        if ldr and ld != ldr and rows > 1:
            raise _abi.DtasError(_abi.EINVAL, f"{name}: both residuals must have the same row stride")
        ldr = ld
    fused = res1 is not None or _ACTS[act] != _abi.ACT_NONE or out.dtype == torch.float32
    return _ACTS[act], (_abi.F32 if out.dtype == torch.float32 else _abi.F16), ldr, fused


def _ptr(t):
    return t.data_ptr() if t is not None else None


def gemv(x, w, out, bias=None, res1=None, res2=None, act=None):
    """out[1, N] = act(x[1, K] @ w[N, K]^T + bias[N]) + res1 + res2; fp16 operands, fp32 accumulation,
    fp16 or fp32 `out` (the fp16 result widened).  bias, res1, res2 and act are optional."""
    tensors = tuple(t for t in (x, w, out, bias, res1, res2) if t is not None)
    dev, st = _check("gemv", *tensors)
    n, k = int(w.shape[0]), int(w.shape[1])
    if w.dim() != 2 or x.numel() != k or out.numel() != n:
        raise _abi.DtasError(_abi.EINVAL, f"gemv: shapes x{tuple(x.shape)} w{tuple(w.shape)} out{tuple(out.shape)}")
    if not (x.dtype == w.dtype == torch.float16):
        raise _abi.DtasError(_abi.EUNSUPPORTED, "gemv: only fp16 operands are implemented")
    act_c, out_c, _, fused = _tail_args("gemv", out, n, 1, bias, res1, res2, act)
    if fused:
        _chk(_lib().dtas_gemv_fused(x.data_ptr(), w.data_ptr(), _ptr(bias), _ptr(res1), _ptr(res2), out.data_ptr(),
                                    n, k, act_c, out_c, _abi.F16, dev, st))
    else:
        _chk(_lib().dtas_gemv(x.data_ptr(), w.data_ptr(), _ptr(bias), out.data_ptr(), n, k, _abi.F16, dev, st))
    return out


def gemm_nt(x, w, out, bias=None, res1=None, res2=None, act=None):
    """out[m, N] = act(x[m, K] @ w[N, K]^T + bias[N]) + res1[m, N] + res2[m, N]; fp16 operands, fp32
    accumulation, fp16 or fp32 `out` (the fp16 result widened).  bias, res1, res2 and act ('gelu')
    are optional: the fused forms of the reference's model workloads.

    `out` may be a column slab of a wider row-major buffer (last-dim stride 1, any row
    stride >= N): a column-sharded rank writes its part of the full output in place.  So may res1 and res2,
    with one row stride; either may be `out` itself.
    """
    dev_t = x.device
    if dev_t.type != "cuda":
        raise _abi.DtasError(_abi.EINVAL, f"gemm: tensors must live on a CUDA device, got {dev_t}")
    m, k = _rows_cols(x, "gemm")
    mo, n = _rows_cols(out, "gemm")
    if w.dim() != 2 or int(w.shape[1]) != k or int(w.shape[0]) != n or mo != m:
        raise _abi.DtasError(_abi.EINVAL, f"gemm: shapes x{tuple(x.shape)} w{tuple(w.shape)} out{tuple(out.shape)}")
    if not (x.dtype == w.dtype == torch.float16):
        raise _abi.DtasError(_abi.EUNSUPPORTED, "gemm: only fp16 operands are implemented")
    if not x.is_contiguous() or not w.is_contiguous():
        raise _abi.DtasError(_abi.EINVAL, "gemm: x and w must be contiguous")
    if out.stride(-1) != 1:
        raise _abi.DtasError(_abi.EINVAL, "gemm: out must have unit stride in its last dim")
    ldy = int(out.stride(-2)) if m > 1 else max(int(out.stride(-2)), n)
    for t in (w, out, bias, res1, res2):
        if t is not None and t.device != dev_t:
            raise _abi.DtasError(_abi.EINVAL, "gemm: tensors on different devices")
    act_c, out_c, ldr, fused = _tail_args("gemm", out, n, m, bias, res1, res2, act)
    dev = dev_t.index if dev_t.index is not None else torch.cuda.current_device()
    st = _raw_stream(dev)
    if fused:
        _chk(_lib().dtas_gemm_nt_fused(x.data_ptr(), w.data_ptr(), _ptr(bias), _ptr(res1), _ptr(res2), out.data_ptr(),
                                       m, n, k, ldy, ldr, act_c, out_c, _abi.F16, dev, st))
    else:
        _chk(_lib().dtas_gemm_nt(x.data_ptr(), w.data_ptr(), _ptr(bias), out.data_ptr(), m, n, k, ldy, _abi.F16,
                                 dev, st))
    return out


def gemm_nt_scatter(x, w, out, peers, bias=None, multicast=0):
    """out[m, N] = x[m, K] @ w[N, K]^T (+ bias), and every stored vector of `out` again into each tensor of
    `peers`: views, on this device, with out's shape and row stride - the place of this rank's column
    slab in the other ranks' gather buffers (peer memory).  One launch; the stores to the peers leave
    from the GEMM's epilogue tile by tile.  Run a barrier across ranks before a gathered buffer is read.
    `multicast`, when not 0, is the address of out's slab in a multicast mapping that covers this GPU's
    buffer and every peer's (PeerGatherBuffer.multicast_address): whole blocks then leave as one
    multimem.st per vector and the NVLink switch stores them into every buffer.
    Raises DtasError(EUNSUPPORTED) below 129 rows (use gemm_nt and peer_push there)."""
    import ctypes
    m, k = _rows_cols(x, "gemm_scatter")
    mo, n = _rows_cols(out, "gemm_scatter")
    if x.device.type != "cuda":
        raise _abi.DtasError(_abi.EINVAL, f"gemm_scatter: tensors must live on a CUDA device, got {x.device}")
    if w.dim() != 2 or int(w.shape[1]) != k or int(w.shape[0]) != n or mo != m:
        raise _abi.DtasError(_abi.EINVAL, f"gemm_scatter: shapes x{tuple(x.shape)} w{tuple(w.shape)} out{tuple(out.shape)}")
    if not (x.dtype == w.dtype == out.dtype == torch.float16) or not x.is_contiguous() or not w.is_contiguous():
        raise _abi.DtasError(_abi.EUNSUPPORTED, "gemm_scatter: contiguous fp16 operands and an fp16 output")
    if out.stride(-1) != 1:
        raise _abi.DtasError(_abi.EINVAL, "gemm_scatter: out must have unit stride in its last dim")
    ldy = int(out.stride(-2)) if m > 1 else max(int(out.stride(-2)), n)
    for p in peers:
        if p.dtype != out.dtype or tuple(p.shape) != tuple(out.shape) or p.stride() != out.stride():
            raise _abi.DtasError(_abi.EINVAL, "gemm_scatter: every peer view must have out's dtype, shape and strides")
    if bias is not None and (bias.dtype != torch.float16 or bias.numel() != n or not bias.is_contiguous()):
        raise _abi.DtasError(_abi.EINVAL, "gemm_scatter: bias must be a contiguous fp16 vector of N elements")
    dev = x.device.index if x.device.index is not None else torch.cuda.current_device()
    ptrs = (ctypes.c_void_p * len(peers))(*[p.data_ptr() for p in peers])
    _chk(_lib().dtas_gemm_nt_scatter_multicast(x.data_ptr(), w.data_ptr(), _ptr(bias), out.data_ptr(), ptrs, len(peers),
                                               int(multicast) or None, m, n, k, ldy, _abi.F16, dev, _raw_stream(dev)))
    return out


# ---- the low-bit path ------------------------------------------------------------------------
# These calls launch kernels of a few microseconds, and every attribute read of a tensor costs a tenth of one: a call
# first asks, in one expression, whether everything is as it should be, and only otherwise goes through the checks that
# say what is not (or that let it pass, as [m, H] beside [1, m, H]).
_IN_CODE = {torch.float16: _abi.F16, torch.float32: _abi.F32}
_NORM_OUT = {torch.float16: _abi.F16, torch.int8: _abi.I8, torch.float8_e4m3fn: _abi.E4M3}
_LOW_CODE = {torch.int8: _abi.I8, torch.float8_e4m3fn: _abi.E4M3}
_W4_IN = {torch.float16: _abi.F16, torch.int8: _abi.I8, torch.float8_e4m3fn: _abi.E4M3}


def _row_scale(name, what, t, rows):
    if t is None or t.dtype != torch.float32 or t.numel() != rows:
        raise _abi.DtasError(_abi.EINVAL, f"{name}: {what} must be an fp32 vector of {rows} elements")


def _check_add_rms_norm(x, res, weight, out, res_out, scale):
    _check("add_rms_norm", *[t for t in (x, res, weight, out, res_out, scale) if t is not None])
    m, h = _rows_cols(x, "add_rms_norm")
    _same_shape("add_rms_norm", x, out)
    for t in (res, res_out):
        if t is not None:
            _same_shape("add_rms_norm", x, t)
            if t.dtype != x.dtype:
                raise _abi.DtasError(_abi.EINVAL, "add_rms_norm: res and res_out must have x's dtype")
    if x.dtype not in _IN_CODE:
        raise _abi.DtasError(_abi.EUNSUPPORTED, f"add_rms_norm: x must be fp16 or fp32, got {x.dtype}")
    if out.dtype not in _NORM_OUT:
        raise _abi.DtasError(_abi.EUNSUPPORTED, f"add_rms_norm: out must be fp16, int8 or float8_e4m3fn, got {out.dtype}")
    if weight.dtype != torch.float16 or weight.numel() != h:
        raise _abi.DtasError(_abi.EINVAL, "add_rms_norm: weight must be fp16 [H]")
    if out.dtype != torch.float16:
        _row_scale("add_rms_norm", "scale", scale, m)


def add_rms_norm(x, res, weight, out, res_out=None, scale=None, eps=1e-6):
    """h = x + res; out = h * rsqrt(mean(h^2, -1) + eps) * weight; res_out = h.  One launch, fp32 arithmetic.

    x and res are fp16 or fp32 of one dtype, weight is fp16 [H]; res may be None (h = x).  `res_out`, when given,
    has x's dtype and may be x or res itself.  `out` is fp16, or int8 / float8_e4m3fn: then `scale`, fp32 [m],
    receives max|row| / Q (Q = 127 or 448) and out holds the row over its scale, rounded to even.  A row
    of zeros gets scale 0; a row with an infinity or a NaN gets a NaN scale."""
    dev, shape, dtype = x.get_device(), x.shape, x.dtype
    code = _NORM_OUT.get(out.dtype)
    if (dev < 0 or code is None or dtype not in _IN_CODE or len(shape) != 2 or out.shape != shape or weight.dtype != torch.float16
            or weight.numel() != shape[1] or weight.get_device() != dev or out.get_device() != dev
            or not (x.is_contiguous() and weight.is_contiguous() and out.is_contiguous())
            or (res is not None and (res.shape != shape or res.dtype != dtype or res.get_device() != dev or not res.is_contiguous()))
            or (res_out is not None and (res_out.shape != shape or res_out.dtype != dtype or res_out.get_device() != dev
                                         or not res_out.is_contiguous()))
            or ((scale is not None or code) and (scale is None or scale.dtype != torch.float32 or scale.numel() != shape[0]
                                                 or scale.get_device() != dev or not scale.is_contiguous()))):
        _check_add_rms_norm(x, res, weight, out, res_out, scale)
    status = (_L or _lib()).dtas_add_rms_norm(
        x.data_ptr(), None if res is None else res.data_ptr(), weight.data_ptr(), out.data_ptr(),
        None if res_out is None else res_out.data_ptr(), None if scale is None else scale.data_ptr(),
        shape[-2], shape[-1], float(eps), _IN_CODE[dtype], code, dev, _raw_stream(dev))
    if status:
        _abi.check(status)
    return out


def _check_quantize(x, out, scale):
    _check("quantize", *[t for t in (x, out, scale) if t is not None])
    _same_shape("quantize", x, out)
    if x.dtype not in _IN_CODE:
        raise _abi.DtasError(_abi.EUNSUPPORTED, f"quantize: x must be fp16 or fp32, got {x.dtype}")
    if out.dtype not in _LOW_CODE:
        raise _abi.DtasError(_abi.EUNSUPPORTED, f"quantize: out must be int8 or float8_e4m3fn, got {out.dtype}")
    _row_scale("quantize", "scale", scale, _rows_cols(x, "quantize")[0])


def quantize(x, out, scale):
    """Rows of x (fp16 or fp32) as int8 or float8_e4m3fn in `out` with one scale each in `scale` (fp32 [m]), as
    add_rms_norm writes them: for activations that no norm precedes, and for the weights of gemm_nt_f8 (a
    scale per output column)."""
    dev, shape, dtype = x.get_device(), x.shape, x.dtype
    code = _LOW_CODE.get(out.dtype)
    if (dev < 0 or code is None or dtype not in _IN_CODE or len(shape) != 2 or out.shape != shape or out.get_device() != dev
            or scale is None or scale.dtype != torch.float32 or scale.numel() != shape[0] or scale.get_device() != dev
            or not (x.is_contiguous() and out.is_contiguous() and scale.is_contiguous())):
        _check_quantize(x, out, scale)
    status = (_L or _lib()).dtas_quantize(x.data_ptr(), out.data_ptr(), scale.data_ptr(), shape[-2], shape[-1], _IN_CODE[dtype],
                                          code, dev, _raw_stream(dev))
    if status:
        _abi.check(status)
    return out


def _check_gemv_w4(x, w, w_scale, out, w_zero, x_scale, bias, res1, res2, act):
    _check("gemv_w4", *[t for t in (x, w, w_scale, out, w_zero, x_scale, bias, res1, res2) if t is not None])
    m, k = _rows_cols(x, "gemv_w4")
    mo, n = _rows_cols(out, "gemv_w4")
    if w.dtype != torch.uint8 or w.dim() != 2 or mo != m or tuple(w.shape) != (n, k // 2) or k % 2:
        raise _abi.DtasError(_abi.EINVAL, f"gemv_w4: shapes x{tuple(x.shape)} w{tuple(w.shape)} out{tuple(out.shape)}; w is uint8 [N, K / 2]")
    groups = int(w_scale.shape[1]) if w_scale.dim() == 2 else 0
    if w_scale.dtype != torch.float16 or groups < 1 or int(w_scale.shape[0]) != n or k % groups:
        raise _abi.DtasError(_abi.EINVAL, f"gemv_w4: w_scale must be fp16 [N, groups] with groups a divisor of K, got {tuple(w_scale.shape)}")
    if w_zero is not None and (w_zero.dtype != torch.uint8 or w_zero.shape != w_scale.shape):
        raise _abi.DtasError(_abi.EINVAL, "gemv_w4: w_zero must be uint8 with w_scale's shape")
    if x.dtype not in _W4_IN:
        raise _abi.DtasError(_abi.EUNSUPPORTED, f"gemv_w4: x must be fp16, int8 or float8_e4m3fn, got {x.dtype}")
    if x.dtype != torch.float16:
        _row_scale("gemv_w4", "x_scale", x_scale, m)
    elif x_scale is not None:
        raise _abi.DtasError(_abi.EINVAL, "gemv_w4: x_scale belongs to an x of 8 bits")
    _tail_args("gemv_w4", out, n, m, bias, res1, res2, act)


def gemv_w4(x, w, w_scale, out, w_zero=None, x_scale=None, bias=None, res1=None, res2=None, act=None):
    """out[m, N] = act(x[m, K] @ W[N, K]^T + bias[N]) + res1 + res2 for up to 16 rows, W in 4 bits:
    W[n, k] = w_scale[n, k // G] * (code - w_zero[n, k // G]).

    `w` is uint8 [N, K / 2], two codes to a byte, the even k in the low half; `w_scale` fp16 [N, K / G] says
    what G is; `w_zero` uint8 of the same shape, 8 everywhere when None (dtas_b200.weights.quantize_w4
    makes all three).  x is fp16, or int8 / float8_e4m3fn with x_scale fp32 [m], as add_rms_norm and
    quantize write them.  out is fp16 or fp32 (the fp16 result widened); the tail is that of gemv, and res1 or res2
    may be `out` itself."""
    dev, xs, os, gs, dtype = x.get_device(), x.shape, out.shape, w_scale.shape, x.dtype
    code = _W4_IN.get(dtype)
    if (dev < 0 or code is None or len(xs) != 2 or len(os) != 2 or len(gs) != 2 or xs[0] != os[0] or os[1] != gs[0]
            or w.shape != (gs[0], xs[1] >> 1) or xs[1] & 1 or gs[1] < 1 or xs[1] % gs[1] or w.dtype != torch.uint8
            or w_scale.dtype != torch.float16 or w.get_device() != dev or w_scale.get_device() != dev or out.get_device() != dev
            or not (x.is_contiguous() and w.is_contiguous() and w_scale.is_contiguous() and out.is_contiguous())
            or (x_scale is None) != (code == _abi.F16)
            or (x_scale is not None and (x_scale.dtype != torch.float32 or x_scale.numel() != xs[0] or x_scale.get_device() != dev
                                         or not x_scale.is_contiguous()))
            or (w_zero is not None and (w_zero.dtype != torch.uint8 or w_zero.shape != gs or w_zero.get_device() != dev
                                        or not w_zero.is_contiguous()))
            or act not in _ACTS or out.dtype not in _IN_CODE
            or (bias is not None and (bias.dtype != torch.float16 or bias.numel() != os[1] or bias.get_device() != dev or not bias.is_contiguous()))
            or (res1 is not None and (res1.dtype != torch.float16 or res1.shape != os or res1.get_device() != dev or not res1.is_contiguous()))
            or (res2 is not None and (res1 is None or res2.dtype != torch.float16 or res2.shape != os or res2.get_device() != dev
                                      or not res2.is_contiguous()))):
        _check_gemv_w4(x, w, w_scale, out, w_zero, x_scale, bias, res1, res2, act)
    status = (_L or _lib()).dtas_gemv_w4(
        x.data_ptr(), None if x_scale is None else x_scale.data_ptr(), w.data_ptr(), w_scale.data_ptr(),
        None if w_zero is None else w_zero.data_ptr(), None if bias is None else bias.data_ptr(),
        None if res1 is None else res1.data_ptr(), None if res2 is None else res2.data_ptr(), out.data_ptr(),
        xs[-2], os[-1], xs[-1], xs[-1] // gs[1], _ACTS[act], code, _IN_CODE[out.dtype], dev, _raw_stream(dev))
    if status:
        _abi.check(status)
    return out


def _check_gemm_nt_f8(x, w, x_scale, w_scale, out, bias, res1, res2, act):
    """-> ldr"""
    dev_t = x.device
    if dev_t.type != "cuda":
        raise _abi.DtasError(_abi.EINVAL, f"gemm_f8: tensors must live on a CUDA device, got {dev_t}")
    m, k = _rows_cols(x, "gemm_f8")
    mo, n = _rows_cols(out, "gemm_f8")
    if w.dim() != 2 or int(w.shape[1]) != k or int(w.shape[0]) != n or mo != m:
        raise _abi.DtasError(_abi.EINVAL, f"gemm_f8: shapes x{tuple(x.shape)} w{tuple(w.shape)} out{tuple(out.shape)}")
    if not (x.dtype == w.dtype == torch.float8_e4m3fn):
        raise _abi.DtasError(_abi.EUNSUPPORTED, "gemm_f8: x and w must be float8_e4m3fn")
    _row_scale("gemm_f8", "x_scale", x_scale, m)
    _row_scale("gemm_f8", "w_scale", w_scale, n)
    for t in (x, w, x_scale, w_scale):
        if not t.is_contiguous():
            raise _abi.DtasError(_abi.EINVAL, "gemm_f8: x, w and the scales must be contiguous")
    if out.stride(-1) != 1:
        raise _abi.DtasError(_abi.EINVAL, "gemm_f8: out must have unit stride in its last dim")
    for t in (w, x_scale, w_scale, out, bias, res1, res2):
        if t is not None and t.device != dev_t:
            raise _abi.DtasError(_abi.EINVAL, "gemm_f8: tensors on different devices")
    return _tail_args("gemm_f8", out, n, m, bias, res1, res2, act)[2]


def gemm_nt_f8(x, w, x_scale, w_scale, out, bias=None, res1=None, res2=None, act=None):
    """out[m, N] = act(x_scale[m] * w_scale[N] * (x[m, K] @ w[N, K]^T) + bias[N]) + res1 + res2 of float8_e4m3fn
    operands with fp32 scales per row of x and per row of w (as quantize writes them); fp32 accumulation,
    fp16 or fp32 `out`.  The tail, residuals and an `out` that are column slabs of wider buffers, and a residual that is
    `out` itself, are those of gemm_nt."""
    dev, xs, ws, os, ldr = x.get_device(), x.shape, w.shape, out.shape, 0
    f8 = torch.float8_e4m3fn
    if (dev < 0 or len(xs) != 2 or len(ws) != 2 or len(os) != 2 or xs[1] != ws[1] or os != (xs[0], ws[0])
            or x.dtype != f8 or w.dtype != f8 or x_scale.dtype != torch.float32 or w_scale.dtype != torch.float32
            or x_scale.numel() != xs[0] or w_scale.numel() != ws[0] or w.get_device() != dev or x_scale.get_device() != dev
            or w_scale.get_device() != dev or out.get_device() != dev
            or not (x.is_contiguous() and w.is_contiguous() and x_scale.is_contiguous() and w_scale.is_contiguous() and out.is_contiguous())
            or act not in _ACTS or out.dtype not in _IN_CODE
            or (bias is not None and (bias.dtype != torch.float16 or bias.numel() != os[1] or bias.get_device() != dev or not bias.is_contiguous()))
            or (res1 is not None and (res1.dtype != torch.float16 or res1.shape != os or res1.get_device() != dev or not res1.is_contiguous()))
            or (res2 is not None and (res1 is None or res2.dtype != torch.float16 or res2.shape != os or res2.get_device() != dev
                                      or not res2.is_contiguous()))):
        ldr = _check_gemm_nt_f8(x, w, x_scale, w_scale, out, bias, res1, res2, act)
    m, n = xs[-2], os[-1]
    ldr = ldr or n
    ldy = n if m == 1 or out.is_contiguous() else out.stride(-2)
    status = (_L or _lib()).dtas_gemm_nt_f8(
        x.data_ptr(), w.data_ptr(), x_scale.data_ptr(), w_scale.data_ptr(), None if bias is None else bias.data_ptr(),
        None if res1 is None else res1.data_ptr(), None if res2 is None else res2.data_ptr(), out.data_ptr(),
        m, n, xs[-1], ldy, ldr, _ACTS[act], _IN_CODE[out.dtype], dev, _raw_stream(dev))
    if status:
        _abi.check(status)
    return out


def poll_status(device=None):
    """Synchronises `device` and raises DtasError(ETIMEOUT) if a bounded device-side wait gave up."""
    if device is None:
        device = torch.cuda.current_device()
    _chk(_lib().dtas_poll_status(int(device)))
