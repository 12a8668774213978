"""Weight-side ConvRot quantisation and the fused INT8 GEMM + dequant (API of tilegen/quant);
4-bit weights with group scales and layers with routed experts beside them."""
from .experts import int8_expert_ffn, quantize_convrot_expert_weights
from .int4 import int4_linear, pack_int4, quantize_convrot_weight_int4, unpack_int4
from .int8_ops import int8_matmul_dequant_chunked
from .rowwise import quantize_rowwise
from .weight import quantize_convrot_weight

__all__ = ["int4_linear", "int8_expert_ffn", "int8_matmul_dequant_chunked", "pack_int4",
           "quantize_convrot_expert_weights", "quantize_convrot_weight", "quantize_convrot_weight_int4",
           "quantize_rowwise", "unpack_int4"]
