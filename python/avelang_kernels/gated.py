"""The gated feed-forward block and the bf16 product's gradients under the reference's ``avelang_kernels`` package name (re-exports)."""
from avelang_b200.bf16_gemm import gemm_transposed_b_backward  # noqa: F401
from avelang_b200.gated import gemm_gated_backward, gemm_gated_transposed_b  # noqa: F401

__all__ = ["gemm_gated_transposed_b", "gemm_gated_backward", "gemm_transposed_b_backward"]
