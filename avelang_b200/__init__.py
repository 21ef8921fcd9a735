"""B200-native block-scaled FP4 GEMM + activation quantise behind the avelang operator convention, and next to them
products on 8-bit integers, the gated feed-forward block and the gradients of the bf16 products."""
from .bf16_gemm import gemm_transposed_b_backward  # noqa: F401
from .fp4_gemm import (  # noqa: F401
    GEMM_1CTA_N128,
    GEMM_1CTA_N256,
    GEMM_2CTA_N128,
    GEMM_2CTA_N192,
    GEMM_2CTA_N256,
    GEMM_AUTO,
    GEMM_SKINNY,
    MXFP4,
    NVFP4,
    SF_ROW_MAJOR,
    SF_TILED,
    Fp4Operand,
    check_device_status,
    gemm_mxfp4_transposed_b,
    gemm_nvfp4_transposed_b,
    gemm_quantized_out_transposed_b,
    linear_mxfp4_decode,
    linear_nvfp4_decode,
    make_operand,
    pack_weight_tiles,
    quantize_mxfp4,
    quantize_nvfp4,
    to_tiled,
)
from .gated import gemm_gated_backward, gemm_gated_transposed_b  # noqa: F401
from .int8_gemm import (  # noqa: F401
    Int8Operand,
    gemm_int8_gated_transposed_b,
    gemm_int8_transposed_b,
    quantize_int8,
)

__all__ = [
    "Fp4Operand", "quantize_nvfp4", "quantize_mxfp4", "gemm_nvfp4_transposed_b", "gemm_mxfp4_transposed_b",
    "gemm_quantized_out_transposed_b", "linear_nvfp4_decode", "linear_mxfp4_decode", "make_operand", "pack_weight_tiles", "to_tiled", "check_device_status", "NVFP4", "MXFP4", "SF_ROW_MAJOR", "SF_TILED",
    "GEMM_AUTO", "GEMM_1CTA_N128", "GEMM_1CTA_N256", "GEMM_2CTA_N256", "GEMM_2CTA_N128", "GEMM_2CTA_N192", "GEMM_SKINNY",
    "Int8Operand", "quantize_int8", "gemm_int8_transposed_b", "gemm_int8_gated_transposed_b",
    "gemm_gated_transposed_b", "gemm_gated_backward", "gemm_transposed_b_backward",
]
