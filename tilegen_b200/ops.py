"""Torch-facing wrappers over the C ABI, plus their ``torch.library`` custom ops.

``rotate_quant``, ``quantize_act`` and ``int8_gemm_dequant`` allocate their outputs with torch's
caching allocator and enqueue the sm_100a kernels on the current stream of the
input's device.  They never fall back to another implementation: an input the
kernels do not handle raises ``ValueError``, a CUDA failure raises
``TileGenError``.  ``int8_gemm_dequant`` with one to ``GEMV_MAX_M`` rows runs the
few-row GEMV on the CUDA cores; with up to ``SPLITK_MAX_M`` rows (see
``splitk_route``) the split-K kernel and a cached, self-clearing scratch per
(device, stream); otherwise the tiled tcgen05 kernel.

Beside them stand the linear's other weight forms: ``int4_gemv_dequant`` (4-bit weights
with group scales, few rows) and the routed experts' ``route_experts``,
``int8_grouped_gemm_dequant`` and ``combine_experts``.

The same functions are registered as ``torch.ops.tilegen.rotate_quant``,
``torch.ops.tilegen.quantize_act``, ``torch.ops.tilegen.quantize_ln_mod``,
``torch.ops.tilegen.int8_gemm_dequant``, ``torch.ops.tilegen.int4_gemv_dequant``,
``torch.ops.tilegen.route_experts``, ``torch.ops.tilegen.int8_grouped_gemm_dequant``
and ``torch.ops.tilegen.combine_experts`` (with fake implementations, so they
trace under ``torch.compile``/``torch.export`` as opaque ops).
"""
from __future__ import annotations

import contextlib
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPE_CODE = {
    torch.float32: _lib.TG_DT_F32,
    torch.float16: _lib.TG_DT_F16,
    torch.bfloat16: _lib.TG_DT_BF16,
}
_SUPPORTED_GROUPS = (4, 16, 64, 256)
# input_act names (tilegen/comfyui/backend.py:174) the quantiser applies itself.
FUSED_ACTS = {"gelu_tanh": _lib.TG_ACT_GELU_TANH, "gelu": _lib.TG_ACT_GELU}
# Butterfly orders of the rotation.  "short" (the default): per radix-4
# butterfly S = (a0 + a2) + (a1 + a3) and each output S - 2*a_i in one fma, and
# the codes' rint(v * inv) in one fma for rows without inf/NaN -- codes differ
# from the reference kernel's by one at rounding ties (about 1e-6 of them on
# DiT-like activations; the parity tolerance allows 1e-3), scales by a few
# ulps.  "reference": the reference kernel's left-to-right sums
# (tilegen/kernels/int8_convrot.py:74-77), bit-identical to it.
ROTATION_ORDERS = {"short": 0, "reference": _lib.TG_QUANT_REFERENCE_ORDER}


def _order_flag(fn: str, order: str) -> int:
    if order not in ROTATION_ORDERS:
        raise ValueError(f"{fn}: order must be one of {sorted(ROTATION_ORDERS)}, got {order!r}")
    return ROTATION_ORDERS[order]


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    if t.data_ptr() % 16:
        t = t.clone()
    return t


# The current stream's handle on a device, without making a Stream object (1.2 us
# of a call's ~10) where torch has the accessor its own generated code uses.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda idx: torch.cuda.current_stream(idx).cuda_stream)


# (shape, stride, dtype) -> an uninitialised tensor on the current device, without
# the dispatcher's round (0.7 us where torch.empty takes 1.6), where torch has the
# allocator entry that its own generated code uses.
_fast_empty = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)
# How many dispatch modes are active; without it (None) the dispatcher is not passed by.
_dispatch_modes = getattr(torch._C, "_len_torch_dispatch_stack", None)
_deterministic = getattr(torch._C, "_get_deterministic_algorithms", torch.are_deterministic_algorithms_enabled)
# The current device once CUDA is in use, which an input on a CUDA device shows.
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _allocator(dev: torch.device):
    """(shape, stride, dtype) -> an uninitialised tensor on the CUDA device ``dev``: torch's own call on another device
    than the current one, where a dispatch mode has to see it, and where the deterministic mode fills new memory."""
    if (_fast_empty is not None and _dispatch_modes is not None and dev.index == _current_device()
            and not _dispatch_modes() and not _deterministic()):
        return _fast_empty
    return lambda shape, stride, dtype: torch.empty_strided(shape, stride, dtype=dtype, device=dev)


def _call(func: str, dev: torch.device, *args) -> None:
    L = _lib.lib()
    current = _current_device()
    idx = dev.index if dev.index is not None else current
    stream = _raw_stream(idx)
    if idx != current:
        with torch.cuda.device(idx):
            st = getattr(L, func)(*args, stream)
    else:
        st = getattr(L, func)(*args, stream)
    if st:
        _lib.check(func, st)


def rotate_quant_max_k() -> int:
    return int(_lib.lib().tg_rotate_quant_max_k())


def rotate_quant(x: torch.Tensor, group: int = 256, order: str = "short"):
    """Group-Hadamard rotation + row-wise int8 quantisation of ``x [M, K]``.

    Returns ``(q int8 [M, K], scale fp32 [M])``.  ``x`` must be a CUDA fp16/bf16
    tensor, ``group`` one of 4/16/64/256 and ``K`` a multiple of 256 (at most
    ``rotate_quant_max_k()``).  ``order``: a key of ``ROTATION_ORDERS``.
    """
    flag = _order_flag("rotate_quant", order)
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("rotate_quant: CUDA tensor required")
    if x.ndim != 2:
        raise ValueError(f"rotate_quant: expected 2-D input, got {tuple(x.shape)}")
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"rotate_quant: fp16/bf16 input required, got {x.dtype}")
    if group not in _SUPPORTED_GROUPS:
        raise ValueError(f"rotate_quant: group must be one of {_SUPPORTED_GROUPS}, got {group}")
    m, k = x.shape
    if k % 256:
        raise ValueError(f"rotate_quant: K={k} must be a multiple of 256")
    x = _aligned(x)
    q = torch.empty((m, k), dtype=torch.int8, device=x.device)
    s = torch.empty((m,), dtype=torch.float32, device=x.device)
    if m:
        _call("tg_quantize_act", x.device, x.data_ptr(), _DTYPE_CODE[x.dtype], m, k, int(group),
              _lib.TG_ACT_NONE | flag, q.data_ptr(), s.data_ptr())
    return q, s


def quantize_act(x: torch.Tensor, group: int = 256, act: str | None = None, order: str = "short"):
    """``act`` applied to ``x [M, K]``, then rotate+quantise (``group`` 4..256) or,
    with ``group=1``, the rotation-free row-wise quantisation of
    tilegen/comfyui/backend.py:230-232.  One pass over ``x`` (``tg_quantize_act``).

    ``act``: None/``"none"``, or a name in ``FUSED_ACTS``; the activation is what
    torch's ``F.gelu`` (``approximate="tanh"`` for ``gelu_tanh``) stores for an
    fp16/bf16 tensor.  Returns ``(q int8 [M, K], scale fp32 [M])``.  ``K`` must be
    a multiple of 256 (of 64 for ``group=1``).  ``order``: a key of
    ``ROTATION_ORDERS`` (the row-wise form has no rotation).
    """
    flag = _order_flag("quantize_act", order)
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("quantize_act: CUDA tensor required")
    if x.ndim != 2:
        raise ValueError(f"quantize_act: expected 2-D input, got {tuple(x.shape)}")
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"quantize_act: fp16/bf16 input required, got {x.dtype}")
    if group != 1 and group not in _SUPPORTED_GROUPS:
        raise ValueError(f"quantize_act: group must be 1 or one of {_SUPPORTED_GROUPS}, got {group}")
    if act in (None, "none"):
        code = _lib.TG_ACT_NONE
    elif act in FUSED_ACTS:
        code = FUSED_ACTS[act]
    else:
        raise ValueError(f"quantize_act: activation {act!r} is not one of {sorted(FUSED_ACTS)}")
    m, k = x.shape
    if k % (64 if group == 1 else 256):
        raise ValueError(f"quantize_act: K={k} must be a multiple of {64 if group == 1 else 256}")
    x = _aligned(x)
    q = torch.empty((m, k), dtype=torch.int8, device=x.device)
    s = torch.empty((m,), dtype=torch.float32, device=x.device)
    if m:
        _call("tg_quantize_act", x.device, x.data_ptr(), _DTYPE_CODE[x.dtype], m, k, int(group), code | flag,
              q.data_ptr(), s.data_ptr())
    return q, s


def quantize_ln_mod(x: torch.Tensor, group: int, scale: torch.Tensor, shift: torch.Tensor, eps: float = 1e-6,
                    rows_per_vector: int | None = None):
    """The DiT block's normalisation in front of a projection, fused into the
    quantiser (``tg_quantize_ln_mod``): ``y = LayerNorm(x) * (1 + scale) + shift``
    (LayerNorm without affine, ``eps``), then rotate+quantise ``y`` with ``group``
    (4..256, the short butterfly order), in one pass over ``x`` -- the modulated
    activations are never written to memory.

    ``x``: ``[..., K]`` fp16/bf16 CUDA, flattened to ``[M, K]`` rows.  ``scale`` and
    ``shift``: ``[K]`` (one vector) or ``[S, ..., K]`` (``S`` vectors, e.g. a DiT's
    per-sample ``[B, 1, K]``), converted to ``x``'s dtype; row ``r`` uses vector
    ``r // rows_per_vector`` (default ``M // S``, which must divide evenly).  Each
    of the normalised row, the product and the sum is rounded to ``x``'s dtype as
    torch's separate ops store them; the mean and variance are fp32 sums in a
    fixed order, so codes match ``F.layer_norm`` + the two ops + ``rotate_quant``
    within the parity tolerance, not bit for bit.  Returns ``(q int8 [M, K],
    scale fp32 [M])``.
    """
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("quantize_ln_mod: CUDA tensor required")
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"quantize_ln_mod: fp16/bf16 input required, got {x.dtype}")
    if group not in _SUPPORTED_GROUPS:
        raise ValueError(f"quantize_ln_mod: group must be one of {_SUPPORTED_GROUPS}, got {group}")
    k = x.shape[-1]
    if k % 256:
        raise ValueError(f"quantize_ln_mod: K={k} must be a multiple of 256")
    x2 = _aligned(x.reshape(-1, k))
    m = x2.shape[0]
    vecs = []
    for name, t in (("scale", scale), ("shift", shift)):
        if not isinstance(t, torch.Tensor) or t.shape[-1] != k:
            raise ValueError(f"quantize_ln_mod: {name} must be a tensor whose last dimension is K={k}")
        vecs.append(_aligned(t.to(device=x.device, dtype=x.dtype).reshape(-1, k)))
    sc, sh = vecs
    if sc.shape != sh.shape:
        raise ValueError(f"quantize_ln_mod: scale {tuple(scale.shape)} and shift {tuple(shift.shape)} differ")
    nvec = sc.shape[0]
    if rows_per_vector is None:
        if m % nvec:
            raise ValueError(f"quantize_ln_mod: {m} rows do not split evenly over {nvec} modulation vectors")
        rows_per_vector = max(1, m // nvec)
    rows_per_vector = int(rows_per_vector)
    if rows_per_vector < 1 or nvec < -(-m // rows_per_vector):
        raise ValueError(f"quantize_ln_mod: {nvec} vectors cannot cover {m} rows at {rows_per_vector} a vector")
    q = torch.empty((m, k), dtype=torch.int8, device=x.device)
    s = torch.empty((m,), dtype=torch.float32, device=x.device)
    if m:
        _call("tg_quantize_ln_mod", x.device, x2.data_ptr(), _DTYPE_CODE[x.dtype], m, k, int(group), float(eps),
              sc.data_ptr(), sh.data_ptr(), rows_per_vector, q.data_ptr(), s.data_ptr())
    return q, s


def int8_gemm_dequant(xq: torch.Tensor, xscale: torch.Tensor, wq: torch.Tensor, wscale: torch.Tensor,
                      bias: torch.Tensor | None, out_dtype: torch.dtype, out: torch.Tensor | None = None) -> torch.Tensor:
    """``((float(xq @ wq.T) * xscale[:, None]) * wscale[None, :]) + bias`` as ``out_dtype``.

    ``xq [M, K]`` and ``wq [N, K]`` int8 on the same CUDA device; ``xscale [M]``;
    ``wscale`` scalar or ``[N]``; ``bias [N]`` fp32/fp16/bf16 or None.  ``out``: an
    optional contiguous ``[M, N]`` ``out_dtype`` tensor on that device (16-byte
    aligned) to write into, e.g. this rank's rows of a ``PeerRowGather`` buffer.
    """
    if not (xq.is_cuda and wq.is_cuda):
        raise ValueError("int8_gemm_dequant: CUDA tensors required")
    if xq.dtype != torch.int8 or wq.dtype != torch.int8:
        raise ValueError("int8_gemm_dequant: int8 operands required")
    if xq.ndim != 2 or wq.ndim != 2 or xq.shape[1] != wq.shape[1]:
        raise ValueError(f"int8_gemm_dequant: shapes {tuple(xq.shape)} x {tuple(wq.shape)}^T do not match")
    if out_dtype not in _DTYPE_CODE:
        raise ValueError(f"int8_gemm_dequant: unsupported out_dtype {out_dtype}")
    dev = xq.device
    m, k = xq.shape
    n = wq.shape[0]
    xq = _aligned(xq)
    wq = _aligned(wq.to(dev))
    xs = xscale.to(device=dev, dtype=torch.float32).reshape(-1).contiguous()
    if xs.numel() != m:
        raise ValueError(f"int8_gemm_dequant: xscale has {xs.numel()} elements, expected {m}")
    ws = wscale.to(device=dev, dtype=torch.float32).reshape(-1).contiguous()
    if ws.numel() not in (1, n):
        raise ValueError(f"weight scale must be scalar or length {n}, got {tuple(wscale.shape)}")
    b_ptr, b_code = None, _lib.TG_DT_F32
    if bias is not None:
        b = bias.to(device=dev).reshape(-1)
        if b.dtype not in _DTYPE_CODE:
            b = b.float()
        b = b.contiguous()
        if b.numel() != n:
            raise ValueError(f"int8_gemm_dequant: bias has {b.numel()} elements, expected {n}")
        bias = b
        b_ptr, b_code = b.data_ptr(), _DTYPE_CODE[b.dtype]
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=dev)
    elif (tuple(out.shape) != (m, n) or out.dtype != out_dtype or out.device != dev or not out.is_contiguous()
          or out.data_ptr() % 16):
        raise ValueError(f"int8_gemm_dequant: out must be a contiguous 16-byte aligned [{m}, {n}] {out_dtype} "
                         f"tensor on {dev}")
    if m and gemv_route(m, n, k):
        _call("tg_int8_gemv_dequant", dev, xq.data_ptr(), xs.data_ptr(), wq.data_ptr(), ws.data_ptr(),
              ws.numel(), b_ptr, b_code, m, n, k, _DTYPE_CODE[out_dtype], out.data_ptr())
    elif m and splitk_route(m, n, k):
        work = _splitk_workspace(dev, m, n)
        _call("tg_int8_gemm_dequant_splitk", dev, xq.data_ptr(), xs.data_ptr(), wq.data_ptr(), ws.data_ptr(),
              ws.numel(), b_ptr, b_code, m, n, k, _DTYPE_CODE[out_dtype], out.data_ptr(), work.data_ptr(),
              work.numel())
    elif m:
        _call("tg_int8_gemm_dequant", dev, xq.data_ptr(), xs.data_ptr(), wq.data_ptr(), ws.data_ptr(),
              ws.numel(), b_ptr, b_code, m, n, k, _DTYPE_CODE[out_dtype], out.data_ptr())
    return out


@contextlib.contextmanager
def sm_budget(sms: int):
    """Within the block, the persistent kernels (rotate+quant, the tiled GEMM) size their
    grids for at most ``sms`` SMs (``tg_set_sm_budget``; process-wide, restored on
    exit).  Use it for kernels that run while a collective is in flight on another
    stream, leaving that collective the SMs it occupies, so both proceed at once."""
    L = _lib.lib()
    old = int(L.tg_sm_budget())
    _lib.check("tg_set_sm_budget", L.tg_set_sm_budget(int(sms)))
    try:
        yield
    finally:
        L.tg_set_sm_budget(old)


# Largest M int8_gemm_dequant sends to the few-row GEMV (tg_int8_gemv_dequant,
# at most 4); 0 sends none there.
GEMV_MAX_M = 4


def gemv_route(m: int, n: int, k: int) -> bool:
    """Whether an m x n x k product goes to the few-row GEMV (at most GEMV_MAX_M rows).

    Measured on B200 at the DiT shapes against the split-K kernel, whole linears
    (quantiser + GEMM) replayed from a CUDA graph with L2 flushed before each:
    the GEMV is faster at M <= 2 everywhere (M = 1: qkv 16.0 vs 21.3 us, o_proj
    9.2 vs 11.0, ffn_up 15.4 vs 20.8, ffn_down 15.9 vs 18.9) and at M <= 4 for
    K < 8192; at K = 13824 with 3-4 rows the two are even, and split-K stays.
    """
    return 0 < m <= min(GEMV_MAX_M, 4 if k < 8192 else 2)


# Largest M int8_gemm_dequant sends to the split-K kernel
# (tg_int8_gemm_dequant_splitk); 0 sends every M to the tiled kernel.
SPLITK_MAX_M = 128


def splitk_route(m: int, n: int, k: int) -> bool:
    """Whether an m x n x k product goes to the split-K kernel (at most SPLITK_MAX_M rows).

    Measured on B200 at the DiT shapes against the tiled kernel (whose M <= 128
    tiles give only N/128 CTAs), whole linears replayed from a CUDA graph with
    L2 flushed before each (cold weights, as in a model): split-K is faster for
    M <= 24 everywhere, and up to 128 rows when N <= 8192 or K >= 8192.
    """
    if not 0 < m <= SPLITK_MAX_M:
        return False
    return m <= 24 or n <= 8192 or k >= 8192


# Split-K scratch, one per (device, stream): zero-filled when created and left
# zero by every call, so it is reused as is; it only grows.
_SPLITK_WS: dict[tuple[int, int], torch.Tensor] = {}


def _splitk_workspace(dev: torch.device, m: int, n: int) -> torch.Tensor:
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    key = (idx, torch.cuda.current_stream(idx).cuda_stream)
    need = int(_lib.lib().tg_int8_gemm_dequant_splitk_workspace(m, n))
    ws = _SPLITK_WS.get(key)
    if ws is None or ws.numel() < need:
        # The caching allocator returns 512-byte aligned blocks (256 needed).
        ws = torch.zeros(max(need, 1 << 20), dtype=torch.uint8, device=torch.device("cuda", idx))
        _SPLITK_WS[key] = ws
    return ws


# Most activation rows int4_gemv_dequant takes (TG_INT4_MAX_M); the groups of
# input channels that share a scale; the router's limits.
INT4_MAX_M = 64
INT4_GROUPS = (32, 64, 128, 256)
MAX_EXPERTS = 1024
MAX_TOP_K = 32


def _on(fn: str, name: str, t, dev: torch.device, dtypes, ndim: int) -> None:
    """``t`` is a tensor on ``dev`` of one of ``dtypes`` and of ``ndim`` dimensions, or ValueError."""
    if isinstance(t, torch.Tensor) and t.dtype in dtypes and t.ndim == ndim and t.device == dev:
        return
    if not isinstance(t, torch.Tensor) or t.device != dev:
        raise ValueError(f"{fn}: {name} must be a tensor on {dev}")
    raise ValueError(f"{fn}: {name} must be {ndim}-D of {' / '.join(map(str, dtypes))}, got {tuple(t.shape)} {t.dtype}")


# The level of forward-mode differentiation: without one (-1) no tensor has a tangent.
_dual_level = (lambda: forward_ad._current_level) if hasattr(forward_ad, "_current_level") else (lambda: 0)


def no_gradient(fn: str, *tensors) -> None:
    """The forms for serving have no derivatives: an input that wants a gradient or carries a tangent is refused."""
    wanted = torch.is_grad_enabled()
    dual = _dual_level() >= 0
    if not (wanted or dual):
        return
    for t in tensors:
        if t is not None and (wanted and t.requires_grad or dual and forward_ad.unpack_dual(t).tangent is not None):
            raise ValueError(f"{fn}: no gradient is computed; call it under torch.no_grad() or on detached tensors")


def _out(fn: str, out: torch.Tensor | None, shape: tuple[int, int], dtype: torch.dtype, dev: torch.device,
         align: int = 16) -> torch.Tensor:
    if out is None:
        return _allocator(dev)(shape, (shape[1] or 1, 1), dtype)
    if (tuple(out.shape) != shape or out.dtype != dtype or out.device != dev or not out.is_contiguous()
            or out.data_ptr() % align):
        raise ValueError(f"{fn}: out must be a contiguous {align}-byte aligned {list(shape)} {dtype} tensor on {dev}")
    return out


_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_F32, _I8, _U8, _I32 = (torch.float32,), (torch.int8,), (torch.uint8,), (torch.int32,)


def int4_gemv_dequant(xq: torch.Tensor, xscale: torch.Tensor, w4: torch.Tensor, wscale: torch.Tensor,
                      bias: torch.Tensor | None, out_dtype: torch.dtype,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Few rows of int8 codes times a 4-bit weight with group scales (``tg_int4_gemv_dequant``):
    ``out[m, n] = (sum_g wscale[n, g] * (xq[m, g] . w4[n, g])) * xscale[m] + bias[n]``.

    ``xq [M, K]`` int8 with ``xscale [M]`` as the quantisers return them, ``M`` at
    most ``INT4_MAX_M``; ``w4 [N, K/2]`` uint8 in the layout of
    ``tilegen_b200.quant.pack_int4`` and ``wscale [N, K/group]`` fp32/fp16/bf16 as
    ``quantize_convrot_weight_int4`` returns them (``group``, read off the shapes,
    32, 64, 128 or 256; ``K`` a multiple of 128); ``bias [N]`` or None.  From
    two rows up a row's result does not depend on the others; one row alone is added
    up in another order (another kernel).  ``out``: an optional contiguous
    ``[M, N]`` ``out_dtype`` tensor to write into.
    """
    fn = "int4_gemv_dequant"
    if not isinstance(xq, torch.Tensor) or not xq.is_cuda:
        raise ValueError(f"{fn}: CUDA tensors required")
    dev = xq.device
    _on(fn, "xq", xq, dev, _I8, 2)
    _on(fn, "xscale", xscale, dev, _F32, 1)
    _on(fn, "w4", w4, dev, _U8, 2)
    _on(fn, "wscale", wscale, dev, _FLOATS, 2)
    if out_dtype not in _DTYPE_CODE:
        raise ValueError(f"{fn}: unsupported out_dtype {out_dtype}")
    m, k = xq.shape
    n = w4.shape[0]
    if m > INT4_MAX_M:
        raise ValueError(f"{fn}: {m} rows, at most {INT4_MAX_M}")
    if k % 128 or k == 0 or n == 0 or w4.shape[1] * 2 != k:
        raise ValueError(f"{fn}: w4 {tuple(w4.shape)} does not match K={k} (a multiple of 128, two codes a byte)")
    groups = wscale.shape[1]
    if wscale.shape[0] != n or groups == 0 or k % groups or k // groups not in INT4_GROUPS:
        raise ValueError(f"{fn}: wscale {tuple(wscale.shape)} is not [N, K / group] with group one of {INT4_GROUPS}")
    if xscale.shape[0] != m:
        raise ValueError(f"{fn}: xscale has {xscale.shape[0]} elements, expected {m}")
    b_ptr, b_code = None, _lib.TG_DT_F32
    if bias is not None:
        _on(fn, "bias", bias, dev, _FLOATS, 1)
        if bias.shape[0] != n:
            raise ValueError(f"{fn}: bias has {bias.shape[0]} elements, expected {n}")
        bias = bias.contiguous()
        b_ptr, b_code = bias.data_ptr(), _DTYPE_CODE[bias.dtype]
    no_gradient(fn, xscale, wscale, bias)
    xq, w4, xscale, wscale = _aligned(xq), _aligned(w4), xscale.contiguous(), _aligned(wscale)
    out = _out(fn, out, (m, n), out_dtype, dev, out_dtype.itemsize)
    if m:
        _call("tg_int4_gemv_dequant", dev, xq.data_ptr(), xscale.data_ptr(), w4.data_ptr(), wscale.data_ptr(),
              _DTYPE_CODE[wscale.dtype], k // groups, b_ptr, b_code, m, n, k, _DTYPE_CODE[out_dtype], out.data_ptr())
    return out


class ExpertRoutes(NamedTuple):
    """What ``route_experts`` returns; ``T`` tokens, ``k`` experts each."""

    weights: torch.Tensor  # [T, k] fp32
    ids: torch.Tensor      # [T, k] int32, -1 where a slot is left out
    offsets: torch.Tensor  # [E + 1] int32: expert e's rows are offsets[e] .. offsets[e + 1] - 1
    rows: torch.Tensor     # [T * k] int32: row r's token, -1 behind the last row
    place: torch.Tensor    # [T, k] int32: the row of each slot, -1 where it is left out


def route_experts(logits: torch.Tensor, top_k: int, renormalize: bool = True) -> ExpertRoutes:
    """The router of a layer with routed experts (``tg_route_experts``): of ``logits
    [T, E]`` (fp32/fp16/bf16) each token's ``top_k`` experts -- largest first, equal
    logits by ascending index, NaN above everything -- with their softmax weights
    over the chosen experts (``renormalize``) or over all, and the (token, expert)
    slots sorted by expert, then token.  A slot whose logit is -inf (a closed expert,
    a padded token) is left out.  Nothing is read back to the host: ``offsets`` and
    ``rows`` go to ``int8_grouped_gemm_dequant`` and ``place`` and ``weights`` to
    ``combine_experts`` as they are.
    """
    fn = "route_experts"
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise ValueError(f"{fn}: CUDA tensor required")
    dev = logits.device
    _on(fn, "logits", logits, dev, _FLOATS, 2)
    t, e = logits.shape
    top_k = int(top_k)
    if not 1 <= e <= MAX_EXPERTS:
        raise ValueError(f"{fn}: {e} experts, 1 to {MAX_EXPERTS} are supported")
    if not 1 <= top_k <= min(e, MAX_TOP_K):
        raise ValueError(f"{fn}: top_k={top_k} must be 1 to {min(e, MAX_TOP_K)}")
    if t * top_k > 1 << 30:
        raise ValueError(f"{fn}: {t} tokens of {top_k} experts are too many")
    no_gradient(fn, logits)
    logits = logits.contiguous()
    empty = _allocator(dev)
    slots, stride, i32 = (t, top_k), (top_k, 1), torch.int32
    ids, place, weights = empty(slots, stride, i32), empty(slots, stride, i32), empty(slots, stride, torch.float32)
    offsets, rows = empty((e + 1,), (1,), i32), empty((t * top_k,), (1,), i32)
    need = _lib.lib().tg_route_experts_workspace(t, e)
    work = empty((need,), (1,), torch.uint8) if need else None
    _call("tg_route_experts", dev, logits.data_ptr(), _DTYPE_CODE[logits.dtype], t, e, top_k, 1 if renormalize else 0,
          weights.data_ptr(), ids.data_ptr(), offsets.data_ptr(), rows.data_ptr(), place.data_ptr(),
          work.data_ptr() if need else None, need)
    return ExpertRoutes(weights, ids, offsets, rows, place)


def _expert_scales(fn: str, t, e: int, n: int, dev: torch.device) -> None:
    """``t``: one fp32 scale on ``dev``, or ``[e]``, ``[e, n]`` or ``[e * n]`` of them (dimensions of one aside),
    or ValueError: a transposed one has as many elements."""
    if not isinstance(t, torch.Tensor) or t.device != dev or t.dtype != torch.float32:
        raise ValueError(f"{fn}: wscale must be fp32 on {dev}")
    shape = tuple(t.shape)
    if shape != (e, n) and [d for d in shape if d != 1] not in ([], [d for d in (e, n) if d != 1],
                                                                [d for d in (e,) if d != 1], [e * n]):
        raise ValueError(f"{fn}: wscale is {shape}, expected one scale, {(e,)} or {(e, n)}")


def int8_grouped_gemm_dequant(xq: torch.Tensor, xscale: torch.Tensor, wq: torch.Tensor, wscale: torch.Tensor,
                              bias: torch.Tensor | None, offsets: torch.Tensor, out_dtype: torch.dtype,
                              rows: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``int8_gemm_dequant`` with one weight per expert over ragged groups of rows
    (``tg_int8_grouped_gemm_dequant``): for ``offsets[e] <= r < offsets[e + 1]`` and
    ``a = rows[r]`` (``r`` without ``rows``),
    ``out[r] = ((float(xq[a] @ wq[e].T) * xscale[a]) * wscale[e]) + bias[e]``.

    ``xq [M, K]`` int8, ``xscale [M]``; ``wq [E, N, K]`` int8; ``wscale`` one scale,
    ``[E]`` or ``[E, N]`` fp32; ``bias [E, N]`` or None; ``offsets [E + 1]`` and ``rows
    [R]`` int32, as ``route_experts`` returns them.  ``out``: an optional contiguous
    ``[R, N]`` ``out_dtype`` tensor to write into; rows that no group covers are left
    as they were (uninitialised when ``out`` is not given).  Each row is
    bit-identical to ``int8_gemm_dequant`` with its expert's weight.
    """
    fn = "int8_grouped_gemm_dequant"
    if not isinstance(xq, torch.Tensor) or not xq.is_cuda:
        raise ValueError(f"{fn}: CUDA tensors required")
    dev = xq.device
    _on(fn, "xq", xq, dev, _I8, 2)
    _on(fn, "xscale", xscale, dev, _F32, 1)
    _on(fn, "wq", wq, dev, _I8, 3)
    _on(fn, "offsets", offsets, dev, _I32, 1)
    if out_dtype not in _DTYPE_CODE:
        raise ValueError(f"{fn}: unsupported out_dtype {out_dtype}")
    m, k = xq.shape
    e, n, kw = wq.shape
    if not 1 <= e <= MAX_EXPERTS:
        raise ValueError(f"{fn}: {e} experts, 1 to {MAX_EXPERTS} are supported")
    if kw != k or k == 0 or n == 0:
        raise ValueError(f"{fn}: shapes {tuple(xq.shape)} x {tuple(wq.shape)}^T do not match")
    if offsets.shape[0] != e + 1:
        raise ValueError(f"{fn}: offsets has {offsets.shape[0]} elements, expected {e + 1}")
    if xscale.shape[0] != m:
        raise ValueError(f"{fn}: xscale has {xscale.shape[0]} elements, expected {m}")
    _expert_scales(fn, wscale, e, n, dev)
    b_ptr, b_code = None, _lib.TG_DT_F32
    if bias is not None:
        _on(fn, "bias", bias, dev, _FLOATS, 2)
        if tuple(bias.shape) != (e, n):
            raise ValueError(f"{fn}: bias is {tuple(bias.shape)}, expected {(e, n)}")
        bias = bias.contiguous()
        b_ptr, b_code = bias.data_ptr(), _DTYPE_CODE[bias.dtype]
    r, r_ptr = m, None
    if rows is not None:
        _on(fn, "rows", rows, dev, _I32, 1)
        rows = rows.contiguous()
        r, r_ptr = rows.shape[0], rows.data_ptr()
    no_gradient(fn, xscale, wscale, bias)
    xq, wq = _aligned(xq), _aligned(wq)
    xscale, wscale, offsets = xscale.contiguous(), wscale.contiguous(), offsets.contiguous()
    out = _out(fn, out, (r, n), out_dtype, dev)
    if r:
        need = 0 if rows is None else _lib.lib().tg_int8_grouped_gemm_dequant_workspace(r, e, n, k)
        work = _allocator(dev)((need,), (1,), torch.uint8) if need else None
        _call("tg_int8_grouped_gemm_dequant", dev, xq.data_ptr(), xscale.data_ptr(), m, wq.data_ptr(),
              wscale.data_ptr(), wscale.numel(), b_ptr, b_code, r_ptr, offsets.data_ptr(), r, e, n, k,
              _DTYPE_CODE[out_dtype], out.data_ptr(), work.data_ptr() if need else None, need)
    return out


def combine_experts(y: torch.Tensor, place: torch.Tensor, weights: torch.Tensor,
                    residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Each token's experts' rows added up (``tg_combine_experts``): ``out[t] = sum_j
    weights[t, j] * y[place[t, j]] (+ residual[t])`` in fp32, rounded once to ``y``'s dtype.

    ``y [R, N]`` fp32/fp16/bf16; ``place [T, k]`` int32 and ``weights [T, k]`` fp32 as
    ``route_experts`` returns them (a place outside ``[0, R)`` adds nothing);
    ``residual [T, N]`` of ``y``'s dtype or None.  ``out``: an optional contiguous ``[T,
    N]`` tensor to write into, which may be ``residual`` itself but shares no memory
    with an input otherwise.
    """
    fn = "combine_experts"
    if not isinstance(y, torch.Tensor) or not y.is_cuda:
        raise ValueError(f"{fn}: CUDA tensors required")
    dev = y.device
    _on(fn, "y", y, dev, _FLOATS, 2)
    _on(fn, "place", place, dev, _I32, 2)
    _on(fn, "weights", weights, dev, _F32, 2)
    r, n = y.shape
    t, top_k = place.shape
    if weights.shape != place.shape or not 1 <= top_k <= MAX_TOP_K:
        raise ValueError(f"{fn}: place {tuple(place.shape)} and weights {tuple(weights.shape)} must be [T, k] with k "
                         f"1 to {MAX_TOP_K}")
    if n == 0:
        raise ValueError(f"{fn}: y has no columns")
    if residual is not None:
        _on(fn, "residual", residual, dev, (y.dtype,), 2)
        if tuple(residual.shape) != (t, n):
            raise ValueError(f"{fn}: residual is {tuple(residual.shape)}, expected {(t, n)}")
        residual = residual.contiguous()
    no_gradient(fn, y, weights, residual)
    y, place, weights = y.contiguous(), place.contiguous(), weights.contiguous()
    out = _out(fn, out, (t, n), y.dtype, dev, y.element_size())
    if t:
        _call("tg_combine_experts", dev, y.data_ptr(), _DTYPE_CODE[y.dtype], r, place.data_ptr(), weights.data_ptr(),
              t, top_k, None if residual is None else residual.data_ptr(), n, out.data_ptr())
    return out


# ---------------------------------------------------------------- custom ops
@torch.library.custom_op("tilegen::rotate_quant", mutates_args=())
def _rotate_quant_op(x: torch.Tensor, group: int) -> tuple[torch.Tensor, torch.Tensor]:
    return rotate_quant(x, group)


@_rotate_quant_op.register_fake
def _(x, group):
    return x.new_empty(x.shape, dtype=torch.int8), x.new_empty((x.shape[0],), dtype=torch.float32)


@torch.library.custom_op("tilegen::quantize_act", mutates_args=())
def _quantize_act_op(x: torch.Tensor, group: int, act: str | None) -> tuple[torch.Tensor, torch.Tensor]:
    return quantize_act(x, group, act)


@_quantize_act_op.register_fake
def _(x, group, act):
    return x.new_empty(x.shape, dtype=torch.int8), x.new_empty((x.shape[0],), dtype=torch.float32)


@torch.library.custom_op("tilegen::quantize_ln_mod", mutates_args=())
def _quantize_ln_mod_op(x: torch.Tensor, group: int, scale: torch.Tensor, shift: torch.Tensor,
                        eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    return quantize_ln_mod(x, group, scale, shift, eps)


@_quantize_ln_mod_op.register_fake
def _(x, group, scale, shift, eps):
    m = x.numel() // x.shape[-1]
    return x.new_empty((m, x.shape[-1]), dtype=torch.int8), x.new_empty((m,), dtype=torch.float32)


@torch.library.custom_op("tilegen::int8_gemm_dequant", mutates_args=())
def _int8_gemm_dequant_op(xq: torch.Tensor, xscale: torch.Tensor, wq: torch.Tensor, wscale: torch.Tensor,
                          bias: torch.Tensor | None, out_dtype: torch.dtype) -> torch.Tensor:
    return int8_gemm_dequant(xq, xscale, wq, wscale, bias, out_dtype)


@_int8_gemm_dequant_op.register_fake
def _(xq, xscale, wq, wscale, bias, out_dtype):
    return xq.new_empty((xq.shape[0], wq.shape[0]), dtype=out_dtype)


@torch.library.custom_op("tilegen::int4_gemv_dequant", mutates_args=())
def _int4_gemv_dequant_op(xq: torch.Tensor, xscale: torch.Tensor, w4: torch.Tensor, wscale: torch.Tensor,
                          bias: torch.Tensor | None, out_dtype: torch.dtype) -> torch.Tensor:
    return int4_gemv_dequant(xq, xscale, w4, wscale, bias, out_dtype)


@_int4_gemv_dequant_op.register_fake
def _(xq, xscale, w4, wscale, bias, out_dtype):
    return xq.new_empty((xq.shape[0], w4.shape[0]), dtype=out_dtype)


@torch.library.custom_op("tilegen::route_experts", mutates_args=())
def _route_experts_op(logits: torch.Tensor, top_k: int, renormalize: bool) -> tuple[
        torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return tuple(route_experts(logits, top_k, renormalize))


@_route_experts_op.register_fake
def _(logits, top_k, renormalize):
    t, e = logits.shape
    return (logits.new_empty((t, top_k), dtype=torch.float32), logits.new_empty((t, top_k), dtype=torch.int32),
            logits.new_empty((e + 1,), dtype=torch.int32), logits.new_empty((t * top_k,), dtype=torch.int32),
            logits.new_empty((t, top_k), dtype=torch.int32))


@torch.library.custom_op("tilegen::int8_grouped_gemm_dequant", mutates_args=())
def _int8_grouped_gemm_dequant_op(xq: torch.Tensor, xscale: torch.Tensor, wq: torch.Tensor, wscale: torch.Tensor,
                                  bias: torch.Tensor | None, offsets: torch.Tensor, out_dtype: torch.dtype,
                                  rows: torch.Tensor | None) -> torch.Tensor:
    return int8_grouped_gemm_dequant(xq, xscale, wq, wscale, bias, offsets, out_dtype, rows)


@_int8_grouped_gemm_dequant_op.register_fake
def _(xq, xscale, wq, wscale, bias, offsets, out_dtype, rows):
    return xq.new_empty(((xq if rows is None else rows).shape[0], wq.shape[1]), dtype=out_dtype)


@torch.library.custom_op("tilegen::combine_experts", mutates_args=())
def _combine_experts_op(y: torch.Tensor, place: torch.Tensor, weights: torch.Tensor,
                        residual: torch.Tensor | None) -> torch.Tensor:
    return combine_experts(y, place, weights, residual)


@_combine_experts_op.register_fake
def _(y, place, weights, residual):
    return y.new_empty((place.shape[0], y.shape[1]))
