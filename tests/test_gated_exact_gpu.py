"""GPU tier: the gated block's gradients against the oracle that rounds the inner gradients itself, where a missing block of K shows."""
import pytest
import torch

import avelang_b200 as ave
import dense_oracle as D
import gated_oracle as G

pytestmark = pytest.mark.gpu

ACTS = ["silu", "gelu", "gelu_tanh", "relu", None]


def _randn(dev, rows, cols, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn((rows, cols), generator=g, device=dev) * scale).to(torch.bfloat16)


# whole and cut sums, over two segments that end inside a stage, inside a range and at the end of one; tiles ahead of the first
# product's end; both products beside each other; one row
@pytest.mark.parametrize("m,f,h", [(1, 8, 8), (5, 136, 200), (64, 24, 72), (129, 264, 64), (255, 1000, 136), (300, 1336, 520), (777, 376, 1048), (1025, 72, 2056),
                                   (40, 8200, 64), (8200, 40, 64), (9, 4096, 16), (300, 16392, 72), (8200, 264, 136), (130, 5000, 200),
                                   (8, 2824, 1664), (16, 1664, 1704), (32, 2672, 2736), (520, 1200, 2000), (1003, 2744, 1048), (424, 1488, 528),
                                   (1144, 1040, 216), (8, 80, 120), (1760, 1376, 488), (24, 5432, 2632), (1, 8200, 520), (128, 4096, 2048),
                                   (8, 8200, 1032), (16, 4104, 2056), (64, 4096, 4096), (300, 16320, 72), (300, 16448, 72)])
def test_gradients(cuda_device, m, f, h):
    x, wg, wu = _randn(cuda_device, m, h, 1), _randn(cuda_device, f, h, 2, h ** -0.5), _randn(cuda_device, f, h, 3, h ** -0.5)
    dout, gate, up = (_randn(cuda_device, m, f, s) for s in (4, 5, 6))
    for activation in ACTS:
        want = G.gated_backward(dout, x, wg, wu, gate, up, activation)
        G.check(ave.gemm_gated_backward(dout, x, wg, wu, gate, up, activation=activation), want, f"{activation}")
    G.check(ave.gemm_gated_backward(dout, x, wg, wu, gate, up, activation=None, need_dw=False)[:1], want[:1], "dx alone")
    for g, w in zip(ave.gemm_gated_backward(dout, x, wg, wu, gate, up, activation=None, need_dx=False)[1:], want[1:]):
        D.check(g, w, "dw alone")
    ave.check_device_status(cuda_device)


def test_beyond_two_to_the_31_elements(cuda_device):
    m, f, h = 66000, 32776, 8
    g = torch.Generator(device=cuda_device).manual_seed(0)
    dout, gate, up = (torch.randn((m, f), generator=g, device=cuda_device, dtype=torch.bfloat16) for _ in range(3))
    x, wg, wu = _randn(cuda_device, m, h, 4), _randn(cuda_device, f, h, 5), _randn(cuda_device, f, h, 6)
    dx, dwg, dwu = ave.gemm_gated_backward(dout, x, wg, wu, gate, up)
    for rows in (slice(0, 2), slice(32767, 32770), slice(65534, 65538), slice(m - 2, m)):
        D.check(dx[rows], G.gated_backward(dout[rows], x[rows], wg, wu, gate[rows], up[rows], "silu")[0], f"{rows}")
    for cols in (slice(0, 8), slice(16384, 16392), slice(f - 8, f)):
        want = G.gated_backward(dout[:, cols], x, wg[cols], wu[cols], gate[:, cols], up[:, cols], "silu")
        D.check(dwg[cols], want[1], f"{cols}")
        D.check(dwu[cols], want[2], f"{cols}")
    ave.check_device_status(cuda_device)


def test_relu_against_differences(cuda_device):
    """Gates are odd multiples of 1/8: exact in bf16 and never at relu's kink, so that every difference says something."""
    m, f, h = 20, 24, 16
    g = torch.Generator(device=cuda_device).manual_seed(0)
    x = (torch.randint(-1, 2, (m, h), generator=g, device=cuda_device) / 4).to(torch.bfloat16)
    wg, wu = ((torch.randint(-1, 2, (f, h), generator=g, device=cuda_device)).to(torch.bfloat16) for _ in range(2))
    x[:, 0], wg[:, 0] = 0.125, 1.0
    dout = _randn(cuda_device, m, f, 4)
    _, gate, up = ave.gemm_gated_transposed_b(x, wg, wu, activation="relu", save=True)
    assert torch.equal(gate.double(), x.double() @ wg.double().T) and gate.abs().min() >= 0.125
    assert (gate > 0).any() and (gate < 0).any()
    got = ave.gemm_gated_backward(dout, x, wg, wu, gate, up, activation="relu")
    want = G.gated_backward(dout, x, wg, wu, gate, up, "relu")
    args = [x.double(), wg.double(), wu.double()]
    step = 2.0 ** -10      # exact, and times a weight of 1 nowhere near 1/8

    def loss(*a):
        return (dout.double() * D.act(a[0] @ a[1].T, "relu") * (a[0] @ a[2].T)).sum().item()

    compared = 0
    for which in range(3):
        for i, j in ((0, 0), (3, 5), (19, 15), (11, 2)):
            plus, minus = [t.clone() for t in args], [t.clone() for t in args]
            plus[which][i, j] += step
            minus[which][i, j] -= step
            # quadratic in each argument: the central difference is the derivative, up to 2^-52 of a loss of some thousand, some additions long, over the step: below 1e-9
            slope = (loss(*plus) - loss(*minus)) / (2 * step)
            exact = want[which][0][i, j].item()
            # the inner gradients' own rounding is in `want` and not in the loss
            inner = {0: lambda: D.BF16 * ((dout.double() * up.double()).abs() @ args[1].abs() + (dout.double() * gate.double()).abs() @ args[2].abs()),
                     1: lambda: D.BF16 * ((dout.double() * up.double()).abs().T @ args[0].abs()),
                     2: lambda: D.BF16 * ((dout.double() * gate.double()).abs().T @ args[0].abs())}[which]()[i, j].item()
            assert abs(exact - slope) <= inner + 1e-8 * (1 + abs(slope))
            assert abs(got[which][i, j].item() - slope) <= want[which][1][i, j].item() + inner + 1e-8 * (1 + abs(slope))
            compared += 1
    assert compared == 12
