"""Products on 8-bit integers for sm_100a under the reference's ``avelang_kernels`` package name (re-exports)."""
from avelang_b200.int8_gemm import (  # noqa: F401
    INT8_MAX_K,
    Int8Operand,
    gemm_int8_gated_transposed_b,
    gemm_int8_transposed_b,
    quantize_int8,
)

__all__ = ["Int8Operand", "quantize_int8", "gemm_int8_transposed_b", "gemm_int8_gated_transposed_b", "INT8_MAX_K"]
