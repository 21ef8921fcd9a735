"""Gradients of the gated block with its inner gradients rounded to bf16 where the kernels round them, and bounds that count what is
left: the fp32 sums, the one rounding of the result, and inner values so near to a tie that fp32 may round them the other way.

dense_oracle.gated_backward takes 2^-8 of every inner gradient for that rounding, which over a long sum hides whole blocks of K.
"""
import torch

import dense_oracle as D


def _inner(v, slack):
    """(v rounded to bf16, how far the rounding of anything within `slack` of v may lie from that)"""
    r = v.to(torch.bfloat16).double()
    return r, torch.maximum(((v + slack).to(torch.bfloat16).double() - r).abs(), ((v - slack).to(torch.bfloat16).double() - r).abs())


def inner_gradients(dout, gate, up, activation):
    """((d_gate, slack), (d_up, slack)).  Relative errors of activations and slopes in fp32 are below 2^-15; the slope cancels near its
    zeros, where 2^-20 of |dout up| (1 + |gate|) covers it."""
    d, g, u = dout.double(), gate.double(), up.double()
    dg, du = d * u * D.slope(g, activation), d * D.act(g, activation)
    return _inner(dg, 2.0 ** -15 * dg.abs() + 2.0 ** -20 * (d * u).abs() * (1 + g.abs())), _inner(du, 2.0 ** -15 * du.abs())


def gated_backward(dout, x, wg, wu, gate, up, activation):
    """((dx, bound), (dw_gate, bound), (dw_up, bound))"""
    x, wg, wu = x.double(), wg.double(), wu.double()
    (dg, eg), (du, eu) = inner_gradients(dout, gate, up, activation)
    m, f = dg.shape
    dx = dg @ wg + du @ wu
    results = [(dx, _bound(dx, D.sum_bound(2 * f) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()) + eg @ wg.abs() + eu @ wu.abs()))]
    for inner, slack in ((dg, eg), (du, eu)):
        dw = inner.T @ x
        results.append((dw, _bound(dw, D.sum_bound(m) * (inner.abs().T @ x.abs()) + slack.T @ x.abs())))
    return results


def _bound(value, off):
    """Of a sum that is off by at most `off` before it is rounded: the rounding is relative to |value| + off, which after an inner value
    that went the other way may be many times |value|."""
    return off + D.BF16 * (value.abs() + off)


def check(got, want, what=""):
    """Each element within its bound, and all of them within one rounding in the mean square: at most 2^-8 / sqrt 3 of a value, and a
    quarter more for the sums and for inner values that went the other way."""
    for g, w, name in zip(got, want, ("dx", "dw_gate", "dw_up")):
        D.check(g, w, f"{what} {name}")
        if g.numel() >= 4096:
            assert (g.double() - w[0]).norm() <= 1.25 * 2.0 ** -8 / 3 ** 0.5 * w[0].norm(), f"{what} {name}"
