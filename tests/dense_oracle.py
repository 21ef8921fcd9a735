"""Plain 64-bit forms of the integer, gated and gradient operators, and error bounds for comparing with them.

Bounds count roundings: a rounding to bf16 is off by at most 2^-8 of the value (BF16 carries 1 % on top for the fp32 evaluation of
scales and activations, whose relative errors are below 2^-15); a sum of K products on the tensor cores is off by at most
(K / 16 + 16) 2^-23 of the sum of magnitudes (one fp32 addition per 16 products, at worst truncating, and the
addition of the 16).
"""
import math

import torch

BF16 = 1.01 * 2.0 ** -8


def act(x, name):
    if name == "silu":
        return x * torch.special.expit(x)
    if name == "gelu":
        return x * 0.5 * torch.special.erfc(-x / math.sqrt(2))
    if name == "gelu_tanh":
        return x * torch.special.expit(math.sqrt(8 / math.pi) * (x + 0.044715 * x ** 3))
    return torch.clamp_min(x, 0) if name == "relu" else x


def slope(x, name):
    if name == "silu":
        s = torch.special.expit(x)
        return s + x * s * (1 - s)
    if name == "gelu":
        return 0.5 * torch.special.erfc(-x / math.sqrt(2)) + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        s = torch.special.expit(math.sqrt(8 / math.pi) * (x + 0.044715 * x ** 3))
        return s + x * s * (1 - s) * math.sqrt(8 / math.pi) * (1 + 3 * 0.044715 * x * x)
    return (x > 0).double() if name == "relu" else torch.ones_like(x)


def sum_bound(k):
    return (k / 16 + 16) * 2.0 ** -23


def quantize_int8(x):
    x = x.double()
    top = x.abs().amax(dim=1, keepdim=True)
    top = torch.where(top > 0, top, torch.full_like(top, 127.0))
    return torch.round(x * 127 / top).to(torch.int8), (top / 127).reshape(-1)


def int8_gemm(a, b, bias=None, activation=None):
    """(result, bound) for operands with .values and .scales."""
    z = (a.values.double() @ b.values.double().T) * a.scales.double()[:, None] * b.scales.double()
    size = z.abs()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    y = act(z, activation)
    # the argument is off by 4 fp32 roundings of its terms; no activation here is steeper than 1.13
    return y, BF16 * y.abs() + 1.13 * 4 * 2.0 ** -24 * size


def int8_gated(a, wg, wu, activation):
    sa = a.scales.double()[:, None]
    g = (a.values.double() @ wg.values.double().T) * sa * wg.scales.double()
    u = (a.values.double() @ wu.values.double().T) * sa * wu.scales.double()
    y = act(g, activation) * u
    return y, BF16 * y.abs() + 1.13 * 4 * 2.0 ** -24 * (g * u).abs()


def gated(x, wg, wu, activation):
    """((out, bound), (gate, bound), (up, bound))"""
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.T, x @ wu.T
    eg, eu = sum_bound(x.shape[1]) * (x.abs() @ wg.abs().T), sum_bound(x.shape[1]) * (x.abs() @ wu.abs().T)
    a = act(g, activation)
    y = a * u
    return (y, BF16 * y.abs() + 1.13 * eg * (u.abs() + eu) + a.abs() * eu), (g, BF16 * g.abs() + eg), (u, BF16 * u.abs() + eu)


def gated_backward(dout, x, wg, wu, gate, up, activation):
    """((dx, bound), (dw_gate, bound), (dw_up, bound)); the bounds hold the rounding of both inner gradients as well."""
    d, x, wg, wu, g, u = (t.double() for t in (dout, x, wg, wu, gate, up))
    dg, du = d * u * slope(g, activation), d * act(g, activation)
    m, f = d.shape
    dx, sx = dg @ wg + du @ wu, dg.abs() @ wg.abs() + du.abs() @ wu.abs()
    dwg, sg = dg.T @ x, dg.abs().T @ x.abs()
    dwu, su = du.T @ x, du.abs().T @ x.abs()
    # the fp32 slope itself cancels near its zeros: 2^-20 of |d u| (1 + |g|) covers it
    slack = 2.0 ** -20 * (d * u).abs() * (1 + g.abs())
    return ((dx, BF16 * (dx.abs() + sx) + sum_bound(2 * f) * sx + slack @ wg.abs()),
            (dwg, BF16 * (dwg.abs() + sg) + sum_bound(m) * sg + slack.T @ x.abs()),
            (dwu, BF16 * (dwu.abs() + su) + sum_bound(m) * su))


def product_backward(dout, a, b):
    d, a, b = dout.double(), a.double(), b.double()
    da, db = d @ b, d.T @ a
    return ((da, BF16 * da.abs() + sum_bound(d.shape[1]) * (d.abs() @ b.abs())),
            (db, BF16 * db.abs() + sum_bound(d.shape[0]) * (d.abs().T @ a.abs())))


def check(got, want, what=""):
    ref, bound = want
    assert tuple(got.shape) == tuple(ref.shape), (what, got.shape, ref.shape)
    err = (got.double() - ref).abs()
    bad = ~(err <= bound + 1e-37)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}: "
                           f"got {got[tuple(bad.nonzero()[0])].item()}, want {ref[tuple(bad.nonzero()[0])].item()}")
