"""CPU tier: include/ave_dense.h and the library agree; refusals of the integer, gated and gradient operators."""
import ctypes
import os
import re

import pytest
import torch

import avelang_b200 as ave
from avelang_b200 import _dense, _lib, build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = ctypes.c_void_p(4096)     # never dereferenced: the checks come first


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def _bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def _op(rows, k):
    return ave.Int8Operand(torch.zeros((rows, k), dtype=torch.int8), torch.ones(rows))


def test_declared_symbols_are_exported(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "ave_dense.h")).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(ave_[a-z0-9_]+)\s*\(", text)))
    assert sorted(_lib.DENSE_EXPORTS) == declared
    for name in declared:
        assert hasattr(lib, name)


def test_operators_refuse_host_tensors_and_wrong_types():
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        ave.quantize_int8(_bf16(4, 64))
    with pytest.raises(ValueError, match="x must have dtype torch.bfloat16"):
        ave.quantize_int8(torch.zeros((4, 64)))
    with pytest.raises(ValueError, match="A.values must be a CUDA tensor"):
        ave.gemm_int8_transposed_b(_op(4, 64), _op(8, 64))
    with pytest.raises(ValueError, match="A must be an Int8Operand"):
        ave.gemm_int8_transposed_b(torch.zeros((4, 64), dtype=torch.int8), _op(8, 64))
    with pytest.raises(ValueError, match="activation must be one of"):
        ave.gemm_int8_transposed_b(_op(4, 64), _op(8, 64), activation="tanh")
    with pytest.raises(ValueError, match="activation must be one of"):
        ave.gemm_gated_transposed_b(_bf16(4, 64), _bf16(8, 64), _bf16(8, 64), activation="swish")
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        ave.gemm_gated_transposed_b(_bf16(4, 64), _bf16(8, 64), _bf16(8, 64))
    with pytest.raises(ValueError, match="x must have dtype torch.bfloat16"):
        ave.gemm_gated_backward(_bf16(4, 8), torch.zeros((4, 64)), _bf16(8, 64), _bf16(8, 64), _bf16(4, 8), _bf16(4, 8))
    with pytest.raises(ValueError, match="A must be a CUDA tensor"):
        ave.gemm_transposed_b_backward(_bf16(4, 8), _bf16(4, 64), _bf16(8, 64))


def test_matrix_check():
    cpu = torch.device("cpu")
    wide = _bf16(4, 64)
    assert _dense.matrix(wide, "x", torch.bfloat16, 4, 64, cpu) == 64
    assert _dense.matrix(wide[:, 8:40], "x", torch.bfloat16, None, None, cpu) == 64
    assert _dense.matrix(wide[:1, :24], "x", torch.bfloat16, None, None, cpu) == 24
    assert _dense.matrix(wide[:0], "x", torch.bfloat16, None, None, cpu) == 64
    for bad, match in ((wide[:, 4:36], "16-byte aligned"), (wide.T, "row-major"), (wide[:, ::2], "row-major"), (_bf16(4, 12), "16-byte aligned"),
                       (wide[:1].expand(4, 64), "row-major"), (_bf16(64), "2-D"), (_bf16(2, 4, 8), "2-D"), (wide.float(), "dtype")):
        with pytest.raises(ValueError, match=match):
            _dense.matrix(bad, "x", torch.bfloat16, None, None, cpu)
    with pytest.raises(ValueError, match="must have shape"):
        _dense.matrix(wide, "x", torch.bfloat16, 4, 72, cpu)
    with pytest.raises(ValueError, match="must be on device"):
        _dense.matrix(wide, "x", torch.bfloat16, None, None, torch.device("cuda", 0))
    scales = torch.ones(16)
    _dense.vector(scales[4:12], "s", torch.float32, 8, cpu)
    for bad, match in ((scales[1:9], "16-byte aligned"), (scales[::2], "contiguous"), (scales, "shape"), (scales[:8].double(), "float32")):
        with pytest.raises(ValueError, match=match):
            _dense.vector(bad, "s", torch.float32, 8, cpu)
    with pytest.raises(ValueError, match="positive multiple of 16"):
        _dense.multiple(0, "K", 16, positive=True)
    with pytest.raises(ValueError, match="multiple of 8"):
        _dense.multiple(12, "N", 8)


def _refused(lib, rc, text):
    assert rc == -1, rc
    assert text in lib.ave_fp4_last_error().decode(), lib.ave_fp4_last_error()


def test_c_entries_refuse_before_any_launch(lib):
    q, g = lib.ave_int8_quantize, lib.ave_int8_gemm
    _refused(lib, q(P, 4, 24, 24, P, 32, P, None), "K must be a positive multiple of 16")
    _refused(lib, q(P, 4, 32, 36, P, 32, P, None), "row stride of x")
    _refused(lib, q(P, 4, 32, 32, P, 24, P, None), "row stride of values")
    _refused(lib, q(P, 4, 32, 32, ctypes.c_void_p(4100), 32, P, None), "values is null or not 16-byte aligned")
    _refused(lib, q(None, 4, 32, 32, P, 32, P, None), "x is null")
    _refused(lib, q(P, -1, 32, 32, P, 32, P, None), "size out of range")
    _refused(lib, g(P, 64, P, P, 64, P, None, 0, P, 12, None, 0, 4, 12, 64, None), "N must be a multiple of 8")
    _refused(lib, g(P, 64, P, P, 64, P, None, 5, P, 16, None, 0, 4, 16, 64, None), "unknown activation 5")
    _refused(lib, g(P, 131072, P, P, 131072, P, None, 0, P, 16, None, 0, 4, 16, 131072, None), "at most 131056")
    _refused(lib, g(P, 64, None, P, 64, P, None, 0, P, 16, None, 0, 4, 16, 64, None), "the scales of A")
    _refused(lib, g(P, 64, P, P, 64, P, ctypes.c_void_p(4098), 0, P, 16, None, 0, 4, 16, 64, None), "the bias")
    _refused(lib, g(P, 64, P, P, 64, P, None, 0, P, 20, None, 0, 4, 16, 64, None), "row stride of D")
    _refused(lib, lib.ave_int8_gemm_gated(P, 64, P, P, 64, P, P, 56, P, 4, P, 16, None, 0, 4, 16, 64, None), "row stride of W_up")
    _refused(lib, lib.ave_bf16_gemm_gated(P, 64, P, 64, P, 64, 4, P, 16, P, 16, None, 16, None, 0, 4, 16, 64, None), "kept together")
    _refused(lib, lib.ave_bf16_gemm_gated(P, 64, P, 64, P, 64, 4, P, 16, None, 16, None, 16, None, 0, 4, 16, 60, None), "H must be a positive multiple of 8")
    back = lib.ave_bf16_gated_backward
    assert lib.ave_bf16_gated_backward_workspace_bytes(-1, 16, 64, 1, 1) < 0 and lib.ave_bf16_gemm_backward_workspace_bytes(4, 16, -64, 1, 1) < 0
    ok = [P, 16, P, 64, P, 64, P, 64, P, 16, P, 16, 4, P, 64, P, P, 64]
    _refused(lib, back(*ok[:15], P, None, 64, P, 4096, 4, 16, 64, None), "computed together")
    _refused(lib, back(*ok[:8], P, 12, *ok[10:], P, 4096, 4, 16, 64, None), "row stride of gate")
    _refused(lib, lib.ave_bf16_gemm_backward(P, 16, P, 64, P, 64, P, 60, P, 64, None, 0, 4, 16, 64, None), "row stride of dA")
    _refused(lib, lib.ave_bf16_gemm_backward(P, 16, P, 64, P, 64, P, 64, P, 64, None, 0, 4, 12, 64, None), "N must be a multiple of 8")


def test_calls_before_init_fail_loudly(lib):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present; this checks the no-device path")
    assert lib.ave_int8_quantize(P, 4, 32, 32, P, 32, P, None) != 0
    assert lib.ave_bf16_gemm_backward(P, 16, P, 64, P, 64, P, 64, P, 64, None, 0, 4, 16, 64, None) != 0
    assert lib.ave_fp4_last_error()


def test_operators_are_importable_under_the_reference_package_name():
    import importlib
    import sys

    sys.path.insert(0, os.path.join(ROOT, "python"))
    try:
        i8 = importlib.import_module("avelang_kernels.int8_gemm")
        gated = importlib.import_module("avelang_kernels.gated")
    finally:
        sys.path.remove(os.path.join(ROOT, "python"))
    for name in i8.__all__:
        assert getattr(i8, name) is getattr(ave.int8_gemm, name)
    for name in gated.__all__:
        assert getattr(gated, name) is getattr(ave, name)
