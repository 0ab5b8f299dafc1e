"""Bringing a weight matrix to the 4-bit form that ops.gemv_w4 reads: done once, when weights are loaded.

Plain torch on whatever device the weights are on; the 8-bit form (a scale per row) is what ops.quantize
writes.  No counterpart in the reference."""
import torch

from . import _abi


def _groups(w, group):
    if w.dim() != 2 or group < 1 or w.shape[1] % group or w.shape[1] % 2:
        raise _abi.DtasError(_abi.EINVAL, f"w4: weights [N, K] with an even K that the group size divides, got {tuple(w.shape)} and {group}")
    return w.shape[0], w.shape[1] // group


def quantize_w4(w, group=128, zero_points=False):
    """w [N, K] -> (codes uint8 [N, K / 2], scales fp16 [N, K / group], zeros uint8 of that shape or None).

    Without zero points a group's codes are round(w / s) + 8 with s = max|w| / 7; with them the group's range,
    widened to hold 0, is spread over 0..15.  A group of zeros gets scale 0."""
    n, groups = _groups(w, group)
    v = w.float().view(n, groups, group)
    if zero_points:
        lo, hi = v.amin(-1).clamp(max=0), v.amax(-1).clamp(min=0)
        scale = ((hi - lo) / 15).to(torch.float16)
        step = scale.float()
        zero = torch.where(step > 0, -lo / step, torch.zeros_like(lo)).round().clamp(0, 15)
    else:
        scale = (v.abs().amax(-1) / 7).to(torch.float16)
        step = scale.float()
        zero = torch.full_like(step, 8)
    inv = torch.where(step > 0, 1 / step, torch.zeros_like(step))
    code = ((v * inv[..., None]).round() + zero[..., None]).clamp(0, 15).to(torch.uint8).view(n, -1)
    return pack_w4(code), scale, zero.to(torch.uint8) if zero_points else None


def pack_w4(codes):
    """Codes 0..15, uint8 [N, K] -> [N, K / 2], the even k in the low half of a byte."""
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def dequantize_w4(codes, scale, zero=None, dtype=torch.float16):
    """The matrix that codes, scales and zero points stand for, [N, K]: what a prompt too long for
    ops.gemv_w4 multiplies with through ops.gemm_nt."""
    n, groups = scale.shape
    v = torch.stack((codes & 15, codes >> 4), -1).view(n, groups, -1).float()
    z = 8.0 if zero is None else zero.float()[..., None]
    return ((v - z) * scale.float()[..., None]).view(n, -1).to(dtype)
