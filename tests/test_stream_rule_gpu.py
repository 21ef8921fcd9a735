"""GPU tier: few rows of large weights on either side of what sends them to the streaming kernel, by K and by the number of rows."""
import pytest
import torch

import avelang_b200 as ave
import dense_oracle as D

pytestmark = pytest.mark.gpu


def _ints(dev, rows, k, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return ave.Int8Operand(torch.randint(-127, 128, (rows, k), generator=g, device=dev, dtype=torch.int8),
                           torch.rand((rows,), generator=g, device=dev) * 0.02 / k ** 0.5 + 1e-4)


@pytest.mark.parametrize("k", [8176, 8192, 8208, 12288, 16384, 20480])
def test_integers(cuda_device, k):
    b, c = _ints(cuda_device, 4760, k, 2), _ints(cuda_device, 4760, k, 3)
    for m in (1, 2, 8):
        a = _ints(cuda_device, m, k, m)
        D.check(ave.gemm_int8_transposed_b(a, b, activation="silu"), D.int8_gemm(a, b, None, "silu"), f"{m}")
        D.check(ave.gemm_int8_gated_transposed_b(a, b, c), D.int8_gated(a, b, c, "silu"), f"gated {m}")
    ave.check_device_status(cuda_device)


@pytest.mark.parametrize("h", [4088, 4096, 4104, 6144, 8192, 10240])
def test_bf16(cuda_device, h):
    g = torch.Generator(device=cuda_device).manual_seed(1)
    wg, wu = ((torch.randn((2384, h), generator=g, device=cuda_device) * h ** -0.5).to(torch.bfloat16) for _ in range(2))
    for m in (1, 2, 8):
        x = torch.randn((m, h), generator=g, device=cuda_device).to(torch.bfloat16)
        for got, want in zip(ave.gemm_gated_transposed_b(x, wg, wu, save=True), D.gated(x, wg, wu, "silu")):
            D.check(got, want, f"{m}")
    ave.check_device_status(cuda_device)
