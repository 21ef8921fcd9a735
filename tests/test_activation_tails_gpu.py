"""GPU tier: silu and gelu_tanh of arguments so far below zero that exp(-x) nears the end of fp32, or passes it: the result is
still a normal number, and correct to the one rounding.  Results below the normal range (2^-126) may be 0."""
import pytest
import torch

import avelang_b200 as ave
import dense_oracle as D

pytestmark = pytest.mark.gpu

TINY = 2.0 ** -126
# |x| e^x is 3e-38 at -91; the tanh form's argument of the exponential is -87.9 at -10.03
ARGUMENTS = {"silu": (-91.0, -80.0), "gelu_tanh": (-10.2, -9.0)}


def _gates(activation, dev):
    low, high = ARGUMENTS[activation]
    g = torch.linspace(low, high, 512, dtype=torch.float64).to(torch.bfloat16).to(dev)
    assert (D.act(g.double(), activation).abs() > TINY).sum() > 400
    return g


@pytest.mark.parametrize("up", [1.0, 2.0 ** 100])
@pytest.mark.parametrize("m", [2, 20, 200])
@pytest.mark.parametrize("activation", sorted(ARGUMENTS))
def test_forward(cuda_device, activation, m, up):
    g = _gates(activation, cuda_device)
    f = g.numel()
    wg, wu = (torch.zeros((f, 16), dtype=torch.bfloat16, device=cuda_device) for _ in range(2))
    wg[:, 3], wu[:, 3] = g, up
    x = torch.zeros((m, 16), dtype=torch.bfloat16, device=cuda_device)
    x[:, 3] = 1.0
    want = D.act(g.double(), activation).expand(m, f) * up
    D.check(ave.gemm_gated_transposed_b(x, wg, wu, activation=activation), (want, D.BF16 * want.abs() + TINY * up))


@pytest.mark.parametrize("m", [2, 20, 200])
@pytest.mark.parametrize("activation", sorted(ARGUMENTS))
def test_integers(cuda_device, activation, m):
    g = _gates(activation, cuda_device).float()
    n = g.numel()

    def one(rows, scales):
        values = torch.zeros((rows, 32), dtype=torch.int8, device=cuda_device)
        values[:, 5] = 1
        return ave.Int8Operand(values, scales)

    a, b = one(m, torch.ones(m, device=cuda_device)), one(n, g)
    want = D.act(g.double(), activation).expand(m, n)
    D.check(ave.gemm_int8_transposed_b(a, b, activation=activation), (want, D.BF16 * want.abs() + TINY))
    up = 2.0 ** 100
    D.check(ave.gemm_int8_gated_transposed_b(a, b, one(n, torch.full((n,), up, device=cuda_device)), activation=activation),
            (want * up, D.BF16 * want.abs() * up + TINY * up))


@pytest.mark.parametrize("activation", sorted(ARGUMENTS))
def test_backward(cuda_device, activation):
    g = _gates(activation, cuda_device)
    f = g.numel()
    x = torch.zeros((1, 8), dtype=torch.bfloat16, device=cuda_device)
    x[0, 0] = 1.0      # dW[:, 0] is the row of inner gradients itself
    w = torch.zeros((f, 8), dtype=torch.bfloat16, device=cuda_device)
    d = 2.0 ** 90
    dout, up = torch.full((1, f), d, dtype=torch.bfloat16, device=cuda_device), torch.ones((1, f), dtype=torch.bfloat16, device=cuda_device)
    _, dwg, dwu = ave.gemm_gated_backward(dout, x, w, w, g[None], up, activation=activation)
    value, slope = D.act(g.double(), activation) * d, D.slope(g.double(), activation) * d
    D.check(dwu[:, 0], (value, D.BF16 * value.abs() + TINY * d))
    # s (1 + x (1 - s)) carries s, whose last normal value is 2^-126, times |x| and, in the tanh form, its argument's slope
    D.check(dwg[:, 0], (slope, D.BF16 * slope.abs() + 100 * 20 * TINY * d))
