"""CPU tier: the bounds for the gated block's gradients let fp32 arithmetic pass and a missing block of K not."""
import pytest
import torch

import dense_oracle as D
import gated_oracle as G


def _inputs(m, f, h):
    g = torch.Generator().manual_seed(0)
    bf = torch.bfloat16
    dout, gate, up = (torch.randn((m, f), generator=g).to(bf) for _ in range(3))
    x, wg, wu = torch.randn((m, h), generator=g).to(bf), *((torch.randn((f, h), generator=g) * h ** -0.5).to(bf) for _ in range(2))
    return dout, x, wg, wu, gate, up


def _as_fp32(dout, x, wg, wu, gate, up, activation, leave=()):
    """The same in fp32, with bf16 inner gradients; `leave`: columns of F (dx) or rows of M (dw) left out of the sums."""
    (dg, _), (du, _) = G.inner_gradients(dout, gate, up, activation)
    dg, du, x, wg, wu = (t.float() for t in (dg, du, x, wg, wu))
    f, m = torch.ones(dg.shape[1]), torch.ones(dg.shape[0])
    for axis, lo, hi in leave:
        (f if axis == "f" else m)[lo:hi] = 0.0
    return [t.to(torch.bfloat16) for t in ((dg * f) @ wg + du @ wu, (dg * m[:, None]).T @ x, (du * m[:, None]).T @ x)]


@pytest.mark.parametrize("m,f,h,activation", [(300, 16392, 72, "silu"), (24, 5432, 264, "gelu"), (130, 5000, 200, "gelu_tanh"), (1003, 520, 136, "relu")])
def test_bounds(m, f, h, activation):
    args = _inputs(m, f, h)
    want = G.gated_backward(*args, activation)
    G.check(_as_fp32(*args, activation), want)
    # one K block of 64 missing: in dx the last whole one before the second segment starts, in dw somewhere in the middle
    lo = f // 64 * 64 - 64
    short = _as_fp32(*args, activation, leave=(("f", lo, lo + 64),))
    with pytest.raises(AssertionError, match="dx"):
        G.check(short[:1], want[:1])
    with pytest.raises(AssertionError):
        D.check(short[0], want[0])
    if m >= 128:
        short = _as_fp32(*args, activation, leave=(("m", 64, 128),))
        for i in (1, 2):
            with pytest.raises(AssertionError):
                D.check(short[i], want[i])
