"""Feed-forward layers with routed experts on int8 ConvRot weights.

``quantize_convrot_expert_weights`` quantises a stack of expert weights as
``quantize_convrot_weight`` does one; ``int8_expert_ffn`` is the whole layer: the
router, the rotated quantiser, the grouped int8 products and the combine, with no
value read back to the host, so it can be captured in a CUDA graph.  The
reference's linears have one weight.
"""
from __future__ import annotations

import torch

from .. import ops
from .weight import quantize_convrot_weight


def quantize_convrot_expert_weights(weight: torch.Tensor, group_size: int = 256) -> tuple[torch.Tensor, torch.Tensor]:
    """``weight [E, N, K]`` -> ``(wq [E, N, K] int8, wscale [E, N] fp32)``, each row as ``quantize_convrot_weight``."""
    if weight.ndim != 3:
        raise ValueError(f"weight must be 3D [E,N,K], got {tuple(weight.shape)}")
    e, n, k = weight.shape
    wq, wscale = quantize_convrot_weight(weight.reshape(e * n, k), group_size)
    return wq.view(e, n, k), wscale.view(e, n)


def int8_expert_ffn(x: torch.Tensor, logits: torch.Tensor, up, down, top_k: int, *, act: str | None = "gelu_tanh",
                    group_size: int = 256, renormalize: bool = True, residual: torch.Tensor | None = None) -> torch.Tensor:
    """``sum_j w_j * down_e(act(up_e(x)))`` over each token's ``top_k`` experts (+ ``residual``).

    ``x [..., K]`` fp16/bf16 on a CUDA device; ``logits [..., E]`` the router's; ``up``
    and ``down``: ``(wq, wscale, bias or None)`` with ``wq [E, F, K]`` and ``[E, K, F]`` int8
    rotated by ``group_size``; ``act`` None or a name in ``ops.FUSED_ACTS``, applied
    in the second quantiser's pass; ``residual`` of ``x``'s shape (or its rows ``[T, K]``) and dtype.
    """
    k = x.shape[-1]
    x2 = x.reshape(-1, k)
    if logits.shape[:-1] != x.shape[:-1]:
        raise ValueError(f"logits {tuple(logits.shape)} do not match x {tuple(x.shape)}")
    if down[0].shape[1] != k:
        raise ValueError(f"down projects to {down[0].shape[1]} channels, x has {k}")
    if residual is not None and residual.shape not in (x.shape, x2.shape):
        raise ValueError(f"residual {tuple(residual.shape)} is not of x's shape {tuple(x.shape)}")
    ops.no_gradient("int8_expert_ffn", x, logits, residual)
    routes = ops.route_experts(logits.reshape(-1, logits.shape[-1]), top_k, renormalize)
    xq, xscale = ops.rotate_quant(x2, group_size)
    h = ops.int8_grouped_gemm_dequant(xq, xscale, up[0], up[1], up[2], routes.offsets, x.dtype, rows=routes.rows)
    hq, hscale = ops.quantize_act(h, group_size, act)
    y = ops.int8_grouped_gemm_dequant(hq, hscale, down[0], down[1], down[2], routes.offsets, x.dtype)
    res = None if residual is None else residual.reshape(-1, k)
    return ops.combine_experts(y, routes.place, routes.weights, residual=res).reshape(x.shape)
