"""GPU tier: the C entries of include/ave_dense.h on calls that the Python operators never make, and what they keep on the host."""
import ctypes
import time

import pytest
import torch

import avelang_b200 as ave
from avelang_b200 import _lib

pytestmark = pytest.mark.gpu

M, N, K = 890, 512, 11120      # long sums of few tiles: every product here cuts its sum


def _p(t):
    return ctypes.c_void_p(t.data_ptr())


def _bf16(dev, rows, cols, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn((rows, cols), generator=g, device=dev).to(torch.bfloat16)


@pytest.fixture(scope="module")
def lib(cuda_device):
    return _lib.ensure_init(cuda_device.index)


def _entries(lib, dev):
    """(name, bytes of workspace, results, the call as a function of workspace address and size)"""
    stream = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
    a8, b8 = (torch.randint(-127, 128, (r, K), device=dev, dtype=torch.int8) for r in (M, N))
    sa, sb = torch.ones(M, device=dev), torch.ones(N, device=dev)
    x, w = _bf16(dev, M, K // 2, 1), _bf16(dev, N, K // 2, 2)
    out, keep = torch.empty((M, N), dtype=torch.bfloat16, device=dev), (a8, b8, sa, sb, x, w)
    yield ("ave_int8_gemm", lib.ave_int8_gemm_workspace_bytes(M, N, K), (out,), keep, lambda ws, size: lib.ave_int8_gemm(
        _p(a8), K, _p(sa), _p(b8), K, _p(sb), None, 0, _p(out), N, ws, size, M, N, K, stream))
    yield ("ave_int8_gemm_gated", lib.ave_int8_gemm_gated_workspace_bytes(M, N // 2, K), (out,), keep, lambda ws, size: lib.ave_int8_gemm_gated(
        _p(a8), K, _p(sa), _p(b8), K, _p(sb), _p(b8), K, _p(sb), 4, _p(out), N, ws, size, M, N // 2, K, stream))
    yield ("ave_bf16_gemm_gated", lib.ave_bf16_gemm_gated_workspace_bytes(M, N // 2, K // 2), (out,), keep, lambda ws, size: lib.ave_bf16_gemm_gated(
        _p(x), K // 2, _p(w), K // 2, _p(w), K // 2, 4, _p(out), N, None, 0, None, 0, ws, size, M, N // 2, K // 2, stream))
    f, h = 264, 72
    dd, g, u = (_bf16(dev, M, f, s) for s in (3, 4, 5))
    xx, ww = _bf16(dev, M, h, 6), _bf16(dev, f, h, 7)
    dx, dwg, dwu = (torch.empty((r, h), dtype=torch.bfloat16, device=dev) for r in (M, f, f))
    keep = (dd, g, u, xx, ww)
    yield ("ave_bf16_gated_backward", lib.ave_bf16_gated_backward_workspace_bytes(M, f, h, 1, 1), (dx, dwg, dwu), keep,
           lambda ws, size: lib.ave_bf16_gated_backward(_p(dd), f, _p(xx), h, _p(ww), h, _p(ww), h, _p(g), f, _p(u), f, 4, _p(dx), h, _p(dwg), _p(dwu), h,
                                                        ws, size, M, f, h, stream))
    n, k = 16392, 72
    do, aa, bb = _bf16(dev, 300, n, 8), _bf16(dev, 300, k, 9), _bf16(dev, n, k, 10)
    da, db = (torch.empty((r, k), dtype=torch.bfloat16, device=dev) for r in (300, n))
    keep = (do, aa, bb)
    yield ("ave_bf16_gemm_backward", lib.ave_bf16_gemm_backward_workspace_bytes(300, n, k, 1, 1), (da, db), keep,
           lambda ws, size: lib.ave_bf16_gemm_backward(_p(do), n, _p(aa), k, _p(bb), k, _p(da), k, _p(db), k, ws, size, 300, n, k, stream))


def test_workspaces_too_small_or_misaligned_are_refused(lib, cuda_device):
    """Before anything is launched: the results keep what they held.  The right size works, whatever the workspace held."""
    for name, need, results, keep, call in _entries(lib, cuda_device):
        assert need > 0, name
        ws = torch.full((need + 256,), 255, dtype=torch.uint8, device=cuda_device)      # NaN in every format
        for r in results:
            r.fill_(7.0)
        for address, size in ((None, need), (ws.data_ptr(), need - 1), (ws.data_ptr(), 0), (ws.data_ptr() + 16, need), (ws.data_ptr() + 128, need)):
            assert call(ctypes.c_void_p(address), size) == -1, name
            assert "workspace must be 256-byte aligned and hold" in lib.ave_fp4_last_error().decode()
        assert all((r == 7.0).all() for r in results), name
        assert (ws == 255).all(), name
        assert call(ctypes.c_void_p(ws.data_ptr()), need) == 0, name
        first = [r.clone() for r in results]
        assert all(torch.isfinite(r).all() for r in first), name
        assert (ws[need:] == 255).all(), name
        ws.fill_(0)
        assert call(ctypes.c_void_p(ws.data_ptr()), need) == 0, name
        assert all(torch.equal(p, q) for p, q in zip(first, results)), name
    ave.check_device_status(cuda_device)


def test_empty_sums_write_zeros_and_nothing_beside_them(lib, cuda_device):
    stream = ctypes.c_void_p(torch.cuda.current_stream(cuda_device).cuda_stream)
    f, h, ld = 24, 40, 56
    some = _bf16(cuda_device, f, ld)
    hold = [torch.full((f + 1, ld), 7.0, dtype=torch.bfloat16, device=cuda_device) for _ in range(3)]

    def zeroed(t):
        ok = not t[:f, :h].any() and (t[:f, h:] == 7.0).all() and (t[f:] == 7.0).all()
        t.fill_(7.0)
        return bool(ok)

    def untouched(t):
        return bool((t == 7.0).all())

    q = _p(some)
    dx, dwg, dwu = hold
    back = lib.ave_bf16_gated_backward
    assert back(q, f, q, ld, q, ld, q, ld, q, f, q, f, 4, None, ld, _p(dwg), _p(dwu), ld, None, 0, 0, f, h, stream) == 0
    assert zeroed(dwg) and zeroed(dwu) and untouched(dx)
    assert back(q, 0, q, ld, q, ld, q, ld, q, 0, q, 0, 4, _p(dx), ld, None, None, ld, None, 0, f, 0, h, stream) == 0
    assert zeroed(dx) and untouched(dwg) and untouched(dwu)
    assert back(q, f, q, ld, q, ld, q, ld, q, f, q, f, 4, None, ld, None, None, ld, None, 0, 0, f, h, stream) == 0
    product = lib.ave_bf16_gemm_backward
    assert product(q, f, q, ld, q, ld, None, ld, _p(dwg), ld, None, 0, 0, f, h, stream) == 0
    assert zeroed(dwg) and untouched(dx)
    assert product(q, 0, q, ld, q, ld, _p(dx), ld, None, ld, None, 0, f, 0, h, stream) == 0
    assert zeroed(dx) and untouched(dwg)
    # the row stride of one row does not count, and a stride that rows do not fit into is refused
    assert product(q, 0, q, ld, q, ld, _p(dx), 3, None, ld, None, 0, 1, 0, h, stream) == 0
    assert not dx[0, :h].any() and (dx[0, h:] == 7.0).all() and (dx[1:] == 7.0).all()
    assert product(q, 0, q, ld, q, ld, _p(dx), h - 8, None, ld, None, 0, f, 0, h, stream) == -1


def test_plans_of_both_backward_passes_of_one_size_are_kept(lib, cuda_device):
    """A plan takes several microseconds to find, and a product's and a gated block's of the same three sizes have nothing to do with
    one another: asked for in turn they cost no more than one of them again and again.  (Best of many; planning anew each time is ten
    times the call.)"""
    sizes = (777, 1032, 4104)
    gated, product = lib.ave_bf16_gated_backward_workspace_bytes, lib.ave_bf16_gemm_backward_workspace_bytes

    def best(first, second):
        least = 1e9
        for _ in range(30):
            t = time.perf_counter()
            for _ in range(50):
                first(*sizes, 1, 1)
                second(*sizes, 1, 1)
            least = min(least, time.perf_counter() - t)
        return least

    assert best(gated, product) <= 3 * max(best(gated, gated), best(product, product))
