"""4-bit ConvRot weights with group scales, for linears that are bound by their weight's bytes.

``quantize_convrot_weight_int4`` rotates a weight's rows by the group Hadamard, as
``quantize_convrot_weight`` does, and rounds them to signed 4-bit codes with one
scale for each ``scale_group`` input channels; ``int4_linear`` multiplies rotated and
quantised activations with it.  The packed layout is the one the few-row kernel
reads (``tg_int4_gemv_dequant``): of each 128 codes of a row, byte ``16 t + 4 j + b``
holds code ``32 j + 8 t + b`` in its low and code ``32 j + 8 t + 4 + b`` in its high
half.  The reference has no 4-bit form.
"""
from __future__ import annotations

import torch

from .. import ops
from ..kernels.hadamard import build_hadamard, rotate_by_group

_CODE_MAX = 7  # symmetric codes: -7..7 (the kernel also reads -8)
_F16_STEP = 2.0 ** -24  # between fp16's subnormal numbers, and the smallest of them


def pack_int4(codes: torch.Tensor) -> torch.Tensor:
    """Integer codes in [-8, 7], ``[N, K]`` with ``K`` a multiple of 128 -> uint8 ``[N, K/2]``."""
    if codes.ndim != 2 or codes.shape[1] % 128 or codes.dtype not in (torch.int8, torch.int16, torch.int32, torch.int64):
        raise ValueError(f"pack_int4: integer codes [N, K] with K a multiple of 128 required, got "
                         f"{tuple(codes.shape)} {codes.dtype}")
    n, k = codes.shape
    if codes.numel() and (int(codes.min()) < -8 or int(codes.max()) > 7):
        raise ValueError("pack_int4: a code is outside [-8, 7]")
    # [N, block, j, t, half, b] -> [N, block, t, j, half, b]
    c = codes.view(n, k // 128, 4, 4, 2, 4).permute(0, 1, 3, 2, 4, 5).to(torch.uint8) & 15
    return (c[..., 0, :] | (c[..., 1, :] << 4)).reshape(n, k // 2).contiguous()


def unpack_int4(w4: torch.Tensor) -> torch.Tensor:
    """``pack_int4``'s bytes ``[N, K/2]`` -> int8 codes ``[N, K]``."""
    if w4.ndim != 2 or w4.shape[1] % 64 or w4.dtype != torch.uint8:
        raise ValueError(f"unpack_int4: uint8 [N, K/2] with K a multiple of 128 required, got {tuple(w4.shape)} {w4.dtype}")
    n, half = w4.shape
    c = w4.view(n, half // 64, 4, 4, 4)
    c = torch.stack([c & 15, c >> 4], dim=-2).permute(0, 1, 3, 2, 4, 5).reshape(n, half * 2).to(torch.int8)
    return c - 16 * (c >= 8).to(torch.int8)


def quantize_convrot_weight_int4(weight: torch.Tensor, group_size: int = 256, scale_group: int = 128,
                                 scale_dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotate by group Hadamard + 4-bit codes -> ``(w4 [N, K/2] uint8, wscale [N, K/scale_group])``.

    ``group_size`` is the rotation's (``1``: none), ``scale_group`` the channels that
    share a scale.  A scale is absmax/7 in fp32, rounded to ``scale_dtype``; the codes
    divide by the rounded one.  fp32 and bf16 scales are at least 2^-126.  fp16 scales
    below 2^-14 are rounded up to a multiple of 2^-24, so that no code is clipped; where
    other groups are larger, values up to 2^-25 of a group thus become 0, and a weight
    none of whose values reaches 7 * 2^-24 is refused (fp32 and bf16 scales hold it).
    Done once per weight, in fp32, on the weight's device.
    """
    if weight.ndim != 2:
        raise ValueError(f"weight must be 2D [N,K], got {tuple(weight.shape)}")
    n, k = weight.shape
    if k % 128 or k % scale_group or scale_group not in ops.INT4_GROUPS:
        raise ValueError(f"K={k} must be divisible by 128 and by scale_group={scale_group}, one of {ops.INT4_GROUPS}")
    if k % group_size:
        raise ValueError(f"K={k} must be divisible by group_size={group_size}")
    if scale_dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"unsupported scale_dtype {scale_dtype}")
    w = weight.float()
    if group_size != 1:
        w = rotate_by_group(w, build_hadamard(group_size, w.device, w.dtype), group_size)
    w = w.view(n, k // scale_group, scale_group)
    scale = w.abs().amax(dim=-1) / _CODE_MAX
    if scale_dtype == torch.float16:
        most = scale.amax() if scale.numel() else scale.new_zeros(())
        if bool((most > 0) & (most < _F16_STEP)):
            raise ValueError("the weight is too small for fp16 scales: use fp32 or bf16 ones")
        scale = torch.where(scale < torch.finfo(torch.float16).tiny, torch.ceil(scale / _F16_STEP) * _F16_STEP, scale)
        scale = scale.clamp_min(_F16_STEP)
    else:
        scale = scale.clamp_min(torch.finfo(scale_dtype).tiny)
    scale = scale.to(scale_dtype)
    if not bool(torch.isfinite(scale).all()):
        raise ValueError(f"the weight has values that a {scale_dtype} scale cannot hold")
    codes = torch.round(w / scale.float()[..., None]).clamp_(-_CODE_MAX, _CODE_MAX).to(torch.int8)
    return pack_int4(codes.view(n, k)), scale


def int4_linear(x: torch.Tensor, w4: torch.Tensor, wscale: torch.Tensor, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None, group_size: int = 256,
                input_act: str | None = None) -> torch.Tensor:
    """``input_act(x)`` rotated and quantised row-wise, times a 4-bit weight.

    ``x [..., K]`` fp16/bf16 on a CUDA device; ``group_size`` and ``input_act`` as
    ``ops.quantize_act`` takes them (the rotation must be the weight's).  More rows
    than ``ops.INT4_MAX_M`` go through in blocks of that many, each of which streams
    the weight again: for long prompts an int8 weight is the faster form.  From two
    rows up a row's result depends neither on the others nor on how many there are.
    """
    k = x.shape[-1]
    if k != w4.shape[-1] * 2:
        raise ValueError(f"input and weight inner dimensions differ: {k} != {w4.shape[-1] * 2}")
    ops.no_gradient("int4_linear", x)
    out_dtype = out_dtype or x.dtype
    xq, xscale = ops.quantize_act(x.reshape(-1, k), group_size, input_act)
    m, n = xq.shape[0], w4.shape[0]
    if m <= ops.INT4_MAX_M:
        return ops.int4_gemv_dequant(xq, xscale, w4, wscale, bias, out_dtype).reshape(*x.shape[:-1], n)
    y = torch.empty(m, n, dtype=out_dtype, device=x.device)
    s = 0
    while s < m:
        e = min(s + ops.INT4_MAX_M, m)
        if m - e == 1:  # a last row alone would be added up in another order: it takes one along
            e -= 1
        ops.int4_gemv_dequant(xq[s:e], xscale[s:e], w4, wscale, bias, out_dtype, out=y[s:e])
        s = e
    return y.reshape(*x.shape[:-1], n)
