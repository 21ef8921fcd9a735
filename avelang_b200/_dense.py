"""Argument checks and the launch shared by the integer, gated and gradient operators (include/ave_dense.h).

A call for one token runs for a few microseconds on the GPU, so each check is one expression over the usual case; what is
wrong is worked out only once something is.
"""
from __future__ import annotations

import torch

from . import _lib
from .fp4_gemm import ACTIVATIONS


def activation_code(activation: str | None) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(k for k in ACTIVATIONS if k)}, got {activation!r}.")
    return ACTIVATIONS[activation]


_ALIGNED = {torch.bfloat16: 7, torch.int8: 15}      # elements of 16 bytes, less one


def matrix(t: torch.Tensor, name: str, dtype: torch.dtype, rows: int | None = None, cols: int | None = None,
           device: torch.device | None = None) -> int:
    """Check a row-major matrix (any 16-byte aligned row stride); return its row stride."""
    if t.dtype != dtype:
        raise ValueError(f"{name} must have dtype {dtype}, got {t.dtype}.")
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(t.shape)}.")
    r, c = t.shape
    if (t.is_contiguous() and not c & _ALIGNED[dtype] and not t.data_ptr() & 15 and (rows is None or r == rows)
            and (cols is None or c == cols) and (t.is_cuda if device is None else t.device == device)):
        return c
    if (rows is not None and r != rows) or (cols is not None and c != cols):
        raise ValueError(f"{name} must have shape {(r if rows is None else rows, c if cols is None else cols)}, got {(r, c)}.")
    if device is None:
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor, got device {t.device}.")
    elif t.device != device:
        raise ValueError(f"{name} must be on device {device}, got {t.device}.")
    if r == 0 or c == 0:
        return c
    ld, inner = t.stride()
    if r == 1:
        ld = c
    elif ld < c or ld & _ALIGNED[dtype]:
        inner = 0
    if (inner != 1 and (c > 1 or inner == 0)) or t.data_ptr() & 15:
        raise ValueError(f"{name} must be row-major with a 16-byte aligned row stride and address.")
    return ld


def vector(t: torch.Tensor, name: str, dtype: torch.dtype, n: int, device: torch.device) -> None:
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must be a {dtype} tensor of shape ({n},), got {t.dtype} {tuple(t.shape)}.")
    if t.device != device:
        raise ValueError(f"{name} must be on device {device}, got {t.device}.")
    if not t.is_contiguous() or t.data_ptr() & 15:
        raise ValueError(f"{name} must be contiguous and 16-byte aligned.")


def result(out: torch.Tensor | None, name: str, rows: int, cols: int, device: torch.device) -> tuple[torch.Tensor, int]:
    """A given bf16 result, checked, or a new one, and its row stride."""
    if out is None:
        return torch.empty(rows, cols, dtype=torch.bfloat16, device=device), cols
    return out, matrix(out, name, torch.bfloat16, rows, cols, device)


def multiple(value: int, name: str, of: int, positive: bool = False) -> None:
    if value % of or (positive and value == 0):
        raise ValueError(f"{name} must be a {'positive ' if positive else ''}multiple of {of}, got {value}.")


_functions: dict = {}
_needs: dict = {}         # workspace sizes asked for last; they depend on the entry point, the device and the sizes alone
MIN_CUT_BYTES = 4096      # AVE_DENSE_MIN_CUT_BYTES of include/ave_dense.h: shorter rows of K never need a workspace


def forward_workspace(name: str, device: torch.device, m: int, n: int, k: int, k_bytes: int) -> tuple[torch.Tensor | None, int, int]:
    """Workspace of a forward product; few rows and short K are known to need none."""
    if k_bytes < MIN_CUT_BYTES or m <= 8:
        return None, 0, 0
    return workspace(name, device, m, n, k)


def _function(name: str, dev: int):
    if dev not in _lib._inited or name not in _functions:
        _functions[name] = getattr(_lib.ensure_init(dev), name)
    return _functions[name]


def call(name: str, device: torch.device, *args) -> None:
    """Run an entry point on the current stream of `device`, which becomes the current device for the call."""
    dev = device.index
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return call(name, device, *args)
    rc = _function(name, dev)(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        _lib.check(rc)


def workspace(name: str, device: torch.device, *sizes) -> tuple[torch.Tensor | None, int, int]:
    """What `name`_workspace_bytes asks for, for one call on the current stream: (the tensor to hold on to, its address, its size).

    Allocated anew for every call, so calls on other streams and captured graphs have their own.
    """
    dev = device.index
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return workspace(name, device, *sizes)
    key = (name, dev, sizes)
    need = _needs.get(key)
    if need is None:
        need = _function(name + "_workspace_bytes", dev)(*sizes)
        if need < 0:
            _lib.check(need)
        if len(_needs) >= 256:
            _needs.clear()
        _needs[key] = need
    if need == 0:
        return None, 0, 0
    t = torch.empty(need, dtype=torch.uint8, device=device)
    return t, t.data_ptr(), need
