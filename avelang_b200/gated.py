"""The gated half of a feed-forward block on bf16, and its backward pass.

``gemm_gated_transposed_b(x, W_gate, W_up)`` computes ``act(x @ W_gate.T) * (x @ W_up.T)`` in one kernel;
``gemm_gated_backward`` takes the result's gradient to those of x and of both weights.  Together with
``gemm_pipeline_transposed_b`` and ``gemm_transposed_b_backward`` for the down projection they make a training step:

    h, gate, up = gemm_gated_transposed_b(x, W_gate, W_up, save=True)
    y = gemm_pipeline_transposed_b(h, W_down)
    dh, dW_down = gemm_transposed_b_backward(dy, h, W_down)
    dx, dW_gate, dW_up = gemm_gated_backward(dh, x, W_gate, W_up, gate, up)

Nothing is recorded for autograd.
"""
from __future__ import annotations

import torch

from . import _dense


def _inputs(x: torch.Tensor, W_gate: torch.Tensor, W_up: torch.Tensor) -> tuple[int, int, int]:
    ldx = _dense.matrix(x, "x", torch.bfloat16)
    m, h = x.shape
    ldg = _dense.matrix(W_gate, "W_gate", torch.bfloat16, None, None, x.device)
    f = W_gate.shape[0]
    if W_gate.shape[1] != h:
        raise ValueError(f"x and W_gate must share H, got {h} and {W_gate.shape[1]}.")
    ldu = _dense.matrix(W_up, "W_up", torch.bfloat16, f, h, x.device)
    _dense.multiple(f, "F", 8)
    _dense.multiple(h, "H", 8, positive=True)
    return ldx, ldg, ldu


def gemm_gated_transposed_b(x: torch.Tensor, W_gate: torch.Tensor, W_up: torch.Tensor, out: torch.Tensor | None = None,
                            activation: str | None = "silu", save: bool = False
                            ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``out = act(x @ W_gate.T) * (x @ W_up.T)`` for bf16 x (M, H) and W_gate, W_up (F, H); (M, F) bf16.

    Sums, activation ("silu", "gelu", "gelu_tanh", "relu" or None) and product are fp32, rounded once.  ``save=True`` returns
    ``(out, gate, up)`` with the two products as bf16 (M, F), which gemm_gated_backward takes.  H and F must be multiples of 8,
    M is free.  ``out`` may be a column block of a wider matrix; it may not overlap an operand.
    """
    act = _dense.activation_code(activation)
    ldx, ldg, ldu = _inputs(x, W_gate, W_up)
    m, h = x.shape
    f = W_gate.shape[0]
    out, ldd = _dense.result(out, "out", m, f, x.device)
    gate = up = None
    if save:
        gate = torch.empty(m, f, dtype=torch.bfloat16, device=x.device)
        up = torch.empty(m, f, dtype=torch.bfloat16, device=x.device)
    if m and f:
        hold, workspace, need = _dense.forward_workspace("ave_bf16_gemm_gated", x.device, m, f, h, 2 * h)
        _dense.call("ave_bf16_gemm_gated", x.device, x.data_ptr(), ldx, W_gate.data_ptr(), ldg, W_up.data_ptr(), ldu, act,
                    out.data_ptr(), ldd, gate.data_ptr() if save else None, f, up.data_ptr() if save else None, f,
                    workspace, need, m, f, h)
    return (out, gate, up) if save else out


def gemm_gated_backward(dout: torch.Tensor, x: torch.Tensor, W_gate: torch.Tensor, W_up: torch.Tensor, gate: torch.Tensor,
                        up: torch.Tensor, activation: str | None = "silu", need_dx: bool = True, need_dw: bool = True
                        ) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """``(dx, dW_gate, dW_up)`` of gemm_gated_transposed_b from ``dout`` (M, F) and the kept ``gate`` and ``up`` (M, F).

    With d_gate = dout * up * act'(gate) and d_up = dout * act(gate), rounded to bf16:
    ``dx = d_gate @ W_gate + d_up @ W_up``, ``dW_gate = d_gate.T @ x``, ``dW_up = d_up.T @ x``, each summed in fp32 and
    rounded to bf16 once.  relu has slope 0 at 0.  ``need_dx=False`` / ``need_dw=False`` leave those products out and
    return None in their place.
    """
    act = _dense.activation_code(activation)
    ldx, ldg, ldu = _inputs(x, W_gate, W_up)
    m, h = x.shape
    f = W_gate.shape[0]
    dev = x.device
    ld = [_dense.matrix(t, name, torch.bfloat16, m, f, dev) for t, name in ((dout, "dout"), (gate, "gate"), (up, "up"))]
    dx = torch.empty(m, h, dtype=torch.bfloat16, device=dev) if need_dx else None
    dw = torch.empty(2, f, h, dtype=torch.bfloat16, device=dev) if need_dw else None
    dw_gate, dw_up = dw.unbind(0) if need_dw else (None, None)
    if not (need_dx or need_dw):
        return dx, dw_gate, dw_up
    if m and f:
        hold, workspace, need = _dense.workspace("ave_bf16_gated_backward", dev, m, f, h, need_dx, need_dw)
        _dense.call("ave_bf16_gated_backward", dev, dout.data_ptr(), ld[0], x.data_ptr(), ldx, W_gate.data_ptr(), ldg, W_up.data_ptr(), ldu,
                    gate.data_ptr(), ld[1], up.data_ptr(), ld[2], act, dx.data_ptr() if need_dx else None, h,
                    dw_gate.data_ptr() if need_dw else None, dw_up.data_ptr() if need_dw else None, h, workspace, need, m, f, h)
    else:      # an empty sum
        for d in (dx, dw):
            if d is not None:
                d.zero_()
    return dx, dw_gate, dw_up
