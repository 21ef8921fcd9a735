"""Products on 8-bit integers with a scale for each token and each channel, in the framework's operator convention.

* ``quantize_int8(x)`` -> ``Int8Operand``: rows of a bf16 matrix (a token's activations, an output channel's weights) as
  signed 8-bit integers with one fp32 scale per row;
* ``gemm_int8_transposed_b(A, B)``: ``A @ B.T`` of two such operands, bias and activation fused;
* ``gemm_int8_gated_transposed_b(A, W_gate, W_up)``: ``act(A @ W_gate.T) * (A @ W_up.T)`` in one kernel.

As everywhere here: arguments are checked with ``ValueError`` before anything is launched, results are allocated only when not given,
launches are asynchronous on torch's current stream of the operands' device, and nothing is recorded for autograd.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _dense

INT8_MAX_K = 131056      # the 32-bit sums cannot overflow up to here


@dataclass
class Int8Operand:
    """A (rows, k) matrix as integers: element (r, c) is ``values[r, c] * scales[r]``.

    values  int8 (rows, k), K contiguous, the row stride a multiple of 16
    scales  fp32 (rows,)
    """

    values: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self) -> tuple[int, int]:
        return tuple(self.values.shape)

    @property
    def rows(self) -> int:
        return self.values.shape[0]

    @property
    def k(self) -> int:
        return self.values.shape[1]

    @property
    def device(self) -> torch.device:
        return self.values.device


def quantize_int8(x: torch.Tensor, out: Int8Operand | None = None) -> Int8Operand:
    """bf16 (rows, K) -> integers: per row, scale = max|x| / 127 and values = round(127 x / max|x|), ties to even, exactly.

    A row of zeros has scale 1; a row holding an infinity or NaN has scale NaN (all of its products are NaN).
    K must be a multiple of 16; x may be a column block of a wider matrix.  ``out``: an operand of the same shape to overwrite.
    """
    ldx = _dense.matrix(x, "x", torch.bfloat16)
    rows, k = x.shape
    _dense.multiple(k, "K", 16, positive=True)
    if out is None:
        out = Int8Operand(torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format),
                          torch.empty(rows, dtype=torch.float32, device=x.device))
        ldv = k
    else:
        ldv = _operand(out, "out", x.device, rows)
        if out.k != k:
            raise ValueError(f"out must have shape {(rows, k)}, got {out.shape}.")
    if rows:
        _dense.call("ave_int8_quantize", x.device, x.data_ptr(), rows, k, ldx, out.values.data_ptr(), ldv, out.scales.data_ptr())
    return out


def _operand(op: Int8Operand, name: str, device: torch.device | None = None, rows: int | None = None, k: int | None = None) -> int:
    """Check an operand; return its row stride."""
    if not isinstance(op, Int8Operand):
        raise ValueError(f"{name} must be an Int8Operand, got {type(op).__name__}.")
    values = op.values
    ld = _dense.matrix(values, name + ".values", torch.int8, rows, None, device)
    r, c = values.shape
    if k is not None and c != k:
        raise ValueError(f"A and {name} must share K, got {k} and {c}.")
    _dense.vector(op.scales, name + ".scales", torch.float32, r, device or values.device)
    return ld


def _check_k(k: int) -> None:
    _dense.multiple(k, "K", 16, positive=True)
    if k > INT8_MAX_K:
        raise ValueError(f"K must be at most {INT8_MAX_K} (32-bit sums), got {k}.")


def gemm_int8_transposed_b(A: Int8Operand, B: Int8Operand, out: torch.Tensor | None = None,
                           bias: torch.Tensor | None = None, activation: str | None = None) -> torch.Tensor:
    """``out = act(A @ B.T + bias)`` for integer operands A (M, K) and B (N, K), bf16 out.

    The integer sums are exact; scales, ``bias`` ((N,) bf16) and ``activation`` ("relu", "gelu", "gelu_tanh", "silu") are
    applied in fp32 and the result is rounded once.  K must be a multiple of 16 up to 131056, N of 8, M is free.  ``out`` may be a
    column block of a wider matrix; it may not overlap an operand.
    """
    act = _dense.activation_code(activation)
    lda = _operand(A, "A")
    m, k = A.values.shape
    dev = A.values.device
    ldb = _operand(B, "B", dev, None, k)
    n = B.values.shape[0]
    _check_k(k)
    _dense.multiple(n, "N", 8)
    if bias is not None:
        _dense.vector(bias, "bias", torch.bfloat16, n, dev)
    out, ldd = _dense.result(out, "out", m, n, dev)
    if m and n:
        hold, workspace, need = _dense.forward_workspace("ave_int8_gemm", dev, m, n, k, k)
        _dense.call("ave_int8_gemm", dev, A.values.data_ptr(), lda, A.scales.data_ptr(), B.values.data_ptr(), ldb, B.scales.data_ptr(),
                    None if bias is None else bias.data_ptr(), act, out.data_ptr(), ldd,
                    workspace, need, m, n, k)
    return out


def gemm_int8_gated_transposed_b(A: Int8Operand, W_gate: Int8Operand, W_up: Int8Operand, out: torch.Tensor | None = None,
                                 activation: str | None = "silu") -> torch.Tensor:
    """``out = act(A @ W_gate.T) * (A @ W_up.T)`` for integer operands A (M, K) and W_gate, W_up (F, K), bf16 out.

    One pass; the two products never go through memory.  Limits as for gemm_int8_transposed_b (F a multiple of 8).
    """
    act = _dense.activation_code(activation)
    lda = _operand(A, "A")
    m, k = A.values.shape
    dev = A.values.device
    ldg = _operand(W_gate, "W_gate", dev, None, k)
    f = W_gate.values.shape[0]
    ldu = _operand(W_up, "W_up", dev, f, k)
    _check_k(k)
    _dense.multiple(f, "F", 8)
    out, ldd = _dense.result(out, "out", m, f, dev)
    if m and f:
        hold, workspace, need = _dense.forward_workspace("ave_int8_gemm_gated", dev, m, f, k, k)
        _dense.call("ave_int8_gemm_gated", dev, A.values.data_ptr(), lda, A.scales.data_ptr(), W_gate.values.data_ptr(), ldg,
                    W_gate.scales.data_ptr(), W_up.values.data_ptr(), ldu, W_up.scales.data_ptr(), act, out.data_ptr(), ldd,
                    workspace, need, m, f, k)
    return out
