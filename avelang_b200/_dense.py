"""Argument checks and the launch shared by the integer, gated and gradient operators (include/ave_dense.h)."""
from __future__ import annotations

import torch

from . import _lib
from .fp4_gemm import ACTIVATIONS


def activation_code(activation: str | None) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(k for k in ACTIVATIONS if k)}, got {activation!r}.")
    return ACTIVATIONS[activation]


def matrix(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple[int, int] | None = None,
           device: torch.device | None = None) -> int:
    """Check a row-major matrix (any 16-byte aligned row stride); return its row stride."""
    if t.dtype != dtype:
        raise ValueError(f"{name} must have dtype {dtype}, got {t.dtype}.")
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(t.shape)}.")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}.")
    if device is None:
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor, got device {t.device}.")
    elif t.device != device:
        raise ValueError(f"{name} must be on device {device}, got {t.device}.")
    rows, cols = t.shape
    if rows == 0 or cols == 0:
        return cols
    ld, inner = t.stride()
    if (inner != 1 and cols > 1) or (rows > 1 and (ld < cols or ld * t.element_size() % 16)) or t.data_ptr() % 16:
        raise ValueError(f"{name} must be row-major with a 16-byte aligned row stride and address.")
    return ld if rows > 1 else cols


def vector(t: torch.Tensor, name: str, dtype: torch.dtype, n: int, device: torch.device) -> None:
    if t.dtype != dtype or t.shape != (n,):
        raise ValueError(f"{name} must be a {dtype} tensor of shape ({n},), got {t.dtype} {tuple(t.shape)}.")
    if t.device != device:
        raise ValueError(f"{name} must be on device {device}, got {t.device}.")
    if not t.is_contiguous() or t.data_ptr() % 16:
        raise ValueError(f"{name} must be contiguous and 16-byte aligned.")


def result(out: torch.Tensor | None, name: str, shape: tuple[int, int], device: torch.device) -> torch.Tensor:
    """A given bf16 result, checked, or a new one."""
    if out is None:
        return torch.empty(shape, dtype=torch.bfloat16, device=device)
    matrix(out, name, torch.bfloat16, shape, device)
    return out


def multiple(value: int, name: str, of: int, positive: bool = False) -> None:
    if value % of or (positive and value == 0):
        raise ValueError(f"{name} must be a {'positive ' if positive else ''}multiple of {of}, got {value}.")


def call(name: str, device: torch.device, *args) -> None:
    """Run an entry point on the current stream of `device`, which becomes the current device for the call."""
    dev = device.index
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return call(name, device, *args)
    rc = getattr(_lib.ensure_init(dev), name)(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        _lib.check(rc)
