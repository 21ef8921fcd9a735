"""GPU tier: the gated block on bf16, its backward pass and the product's gradients, against 64-bit plain forms."""
import pytest
import torch

import avelang_b200 as ave
import dense_oracle as D
from avelang_b200.bf16_gemm import gemm_pipeline_transposed_b

pytestmark = pytest.mark.gpu

ACTS = ["silu", "gelu", "gelu_tanh", "relu", None]


def _randn(dev, rows, cols, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn((rows, cols), generator=g, device=dev) * scale).to(torch.bfloat16)


def _block(dev, m, f, h):
    return _randn(dev, m, h, 1, 1.0), _randn(dev, f, h, 2, h ** -0.5), _randn(dev, f, h, 3, h ** -0.5)


SHAPES = [(1, 8, 8), (1, 4104, 1024), (5, 136, 200), (8, 24, 2056), (16, 1000, 72), (17, 8, 8), (64, 1000, 136), (128, 520, 264), (129, 264, 64),
          (300, 1336, 520), (513, 2056, 400), (1000, 376, 24)]


@pytest.mark.parametrize("m,f,h", SHAPES)
def test_gated_forward(cuda_device, m, f, h):
    x, wg, wu = _block(cuda_device, m, f, h)
    for activation in ACTS:
        want = D.gated(x, wg, wu, activation)
        out = ave.gemm_gated_transposed_b(x, wg, wu, activation=activation)
        D.check(out, want[0], f"{activation}")
        kept = ave.gemm_gated_transposed_b(x, wg, wu, activation=activation, save=True)
        assert torch.equal(kept[0], out)
        for got, w, what in zip(kept, want, ("out", "gate", "up")):
            D.check(got, w, f"{activation} {what}")
    ave.check_device_status(cuda_device)


@pytest.mark.parametrize("m,f,h", [(1, 8, 8), (5, 136, 200), (64, 24, 72), (129, 264, 64), (255, 1000, 136), (300, 1336, 520), (777, 376, 1048),
                                   (1025, 72, 2056)])
def test_gated_backward(cuda_device, m, f, h):
    x, wg, wu = _block(cuda_device, m, f, h)
    dout = _randn(cuda_device, m, f, 4, 0.1)
    for activation in ACTS:
        _, gate, up = ave.gemm_gated_transposed_b(x, wg, wu, activation=activation, save=True)
        got = ave.gemm_gated_backward(dout, x, wg, wu, gate, up, activation=activation)
        want = D.gated_backward(dout, x, wg, wu, gate, up, activation)
        for g, w, what in zip(got, want, ("dx", "dw_gate", "dw_up")):
            D.check(g, w, f"{activation} {what}")
            if g.numel() >= 4096:
                # two independent roundings, each of at most 2^-8 of a value and so at most 2^-8 / sqrt 3 in the mean square
                assert (g.double() - w[0]).norm() <= 1.25 * 2 ** 0.5 * 2.0 ** -8 / 3 ** 0.5 * w[0].norm()
        again = ave.gemm_gated_backward(dout, x, wg, wu, gate, up, activation=activation)
        assert all(torch.equal(p, q) for p, q in zip(got, again))
    assert ave.gemm_gated_backward(dout, x, wg, wu, gate, up, activation=None, need_dw=False)[1:] == (None, None)
    assert torch.equal(ave.gemm_gated_backward(dout, x, wg, wu, gate, up, activation=None, need_dw=False)[0], got[0])
    dx, dwg, dwu = ave.gemm_gated_backward(dout, x, wg, wu, gate, up, activation=None, need_dx=False)
    assert dx is None and torch.equal(dwg, got[1]) and torch.equal(dwu, got[2])
    ave.check_device_status(cuda_device)


@pytest.mark.parametrize("activation", ACTS)
def test_gradients_against_differences(cuda_device, activation):
    """Inputs whose products are exact in bf16 (quarters up to 4), so that the kept gate and up are the function's own; the
    derivative of sum(dout * f) is taken by central differences in 64 bits."""
    m, f, h = 20, 24, 16
    g = torch.Generator(device=cuda_device).manual_seed(0)
    x = (torch.randint(-1, 2, (m, h), generator=g, device=cuda_device) / 4).to(torch.bfloat16)
    wg, wu = ((torch.randint(-1, 2, (f, h), generator=g, device=cuda_device)).to(torch.bfloat16) for _ in range(2))
    dout = _randn(cuda_device, m, f, 4)
    out, gate, up = ave.gemm_gated_transposed_b(x, wg, wu, activation=activation, save=True)
    assert torch.equal(gate.double(), x.double() @ wg.double().T)
    got = ave.gemm_gated_backward(dout, x, wg, wu, gate, up, activation=activation)
    want = D.gated_backward(dout, x, wg, wu, gate, up, activation)
    args = [x.double(), wg.double(), wu.double()]
    step = 1e-5

    def loss(*a):
        return (dout.double() * D.act(a[0] @ a[1].T, activation) * (a[0] @ a[2].T)).sum().item()

    for which in range(3):
        for i, j in ((0, 0), (3, 5), (19, 15), (11, 2)):
            plus, minus = [t.clone() for t in args], [t.clone() for t in args]
            plus[which][i, j] += step
            minus[which][i, j] -= step
            slope = (loss(*plus) - loss(*minus)) / (2 * step)
            if activation == "relu":
                # at a kink the two one-sided slopes differ: differences say nothing where a gate is exactly 0
                touched = gate[i] if which == 0 else gate[:, i]
                if (touched == 0).any():
                    continue
            assert abs(got[which][i, j].item() - slope) <= want[which][1][i, j].item() + 1e-5 * (1 + abs(slope))


@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (3, 136, 72), (64, 24, 200), (129, 264, 64), (255, 1000, 136), (300, 520, 1336), (777, 1032, 376),
                                   (1025, 72, 2056)])
def test_product_backward(cuda_device, m, n, k):
    a, b, dout = _randn(cuda_device, m, k, 1), _randn(cuda_device, n, k, 2, k ** -0.5), _randn(cuda_device, m, n, 3, 0.1)
    got = ave.gemm_transposed_b_backward(dout, a, b)
    for g, w, what in zip(got, D.product_backward(dout, a, b), ("da", "db")):
        D.check(g, w, what)
    only = ave.gemm_transposed_b_backward(dout, a, b, need_da=False)
    assert only[0] is None and torch.equal(only[1], got[1])
    only = ave.gemm_transposed_b_backward(dout, a, b, need_db=False)
    assert only[1] is None and torch.equal(only[0], got[0])
    ave.check_device_status(cuda_device)


@pytest.mark.parametrize("m", [6, 90, 260])
def test_strided_operands(cuda_device, m):
    f, h = 104, 152
    x, wg, wu = (_randn(cuda_device, r, h + 48, s, 0.2)[:, 8:h + 8] for r, s in ((m, 1), (f, 2), (f, 3)))
    hold = torch.full((m + 2, f + 32), 7.0, dtype=torch.bfloat16, device=cuda_device)
    out = hold[1:m + 1, 16:f + 16]
    assert ave.gemm_gated_transposed_b(x, wg, wu, out=out) is out
    D.check(out, D.gated(x, wg, wu, "silu")[0])
    out.fill_(7.0)
    assert (hold == 7.0).all()
    dout, gate, up = (_randn(cuda_device, m, f + 16, s)[:, :f] for s in (4, 5, 6))
    for g, w in zip(ave.gemm_gated_backward(dout, x, wg, wu, gate, up), D.gated_backward(dout, x, wg, wu, gate, up, "silu")):
        D.check(g, w)
    for g, w in zip(ave.gemm_transposed_b_backward(dout, x, wg), D.product_backward(dout, x, wg)):
        D.check(g, w)


def test_no_rows_and_no_columns(cuda_device):
    x, wg, wu = _block(cuda_device, 4, 16, 24)
    none = x[:0]
    assert ave.gemm_gated_transposed_b(none, wg, wu).shape == (0, 16)
    assert ave.gemm_gated_transposed_b(x, wg[:0], wu[:0]).shape == (4, 0)
    e = torch.empty((0, 16), dtype=torch.bfloat16, device=cuda_device)
    dx, dwg, dwu = ave.gemm_gated_backward(e, none, wg, wu, e, e)
    assert dx.shape == (0, 24) and not dwg.any() and not dwu.any() and dwg.shape == dwu.shape == (16, 24)
    e = torch.empty((4, 0), dtype=torch.bfloat16, device=cuda_device)
    dx, dwg, dwu = ave.gemm_gated_backward(e, x, wg[:0], wu[:0], e, e)
    assert dx.shape == (4, 24) and not dx.any() and dwg.shape == (0, 24)
    da, db = ave.gemm_transposed_b_backward(e, x, wg[:0])
    assert da.shape == (4, 24) and not da.any() and db.shape == (0, 24)


def test_values_that_are_not_finite_stay_in_their_rows(cuda_device):
    m, f, h = 140, 72, 136
    x, wg, wu = _block(cuda_device, m, f, h)
    for rows in (m, 10):
        xi = x[:rows].clone()
        xi[3, 100] = float("nan")
        xi[7, 5] = float("inf")
        out = ave.gemm_gated_transposed_b(xi, wg, wu)
        fine = [r for r in range(rows) if r not in (3, 7)]
        assert torch.isnan(out[3]).all() and torch.isfinite(out[fine]).all()
        assert torch.equal(out[fine], ave.gemm_gated_transposed_b(x[:rows], wg, wu)[fine])
    # gradients: a NaN in one token's dout reaches that token's dx and the weights' gradients, no other token
    dout = _randn(cuda_device, m, f, 4)
    _, gate, up = ave.gemm_gated_transposed_b(x, wg, wu, save=True)
    clean = ave.gemm_gated_backward(dout, x, wg, wu, gate, up)
    dout[m - 1, f - 1] = float("nan")
    dx, dwg, dwu = ave.gemm_gated_backward(dout, x, wg, wu, gate, up)
    assert torch.isnan(dx[m - 1]).all() and torch.equal(dx[:m - 1], clean[0][:m - 1])
    assert torch.isnan(dwg[f - 1]).all() and torch.equal(dwg[:f - 1], clean[1][:f - 1]) and torch.equal(dwu[:f - 1], clean[2][:f - 1])


@pytest.mark.parametrize("activation", ACTS)
def test_far_arguments(cuda_device, activation):
    """Gates over the whole range of bf16: values and slopes keep their limits."""
    g = torch.cat([torch.linspace(-40, 40, 1001), torch.tensor([1e4, -1e4, 1e18, -1e18, 0.0, -0.0, 1e-30])]).to(torch.bfloat16)
    f = g.numel() // 8 * 8
    g = g[-f:].to(cuda_device)[None, :].expand(2, f).contiguous()
    up, dout = torch.ones_like(g), torch.ones_like(g)
    x = torch.zeros((2, 8), dtype=torch.bfloat16, device=cuda_device)
    x[0, 0] = 1.0      # dW[:, 0] is the row of inner gradients itself
    w = torch.zeros((f, 8), dtype=torch.bfloat16, device=cuda_device)
    _, dwg, dwu = ave.gemm_gated_backward(dout, x, w, w, g, up, activation=activation)
    gd = g[0].double()
    # rounded to bf16 twice, the second time without effect; the slope cancels near its zeros, see the oracle
    D.check(dwu[:, 0], (D.act(gd, activation), D.BF16 * D.act(gd, activation).abs() + 1e-30))
    D.check(dwg[:, 0], (D.slope(gd, activation).nan_to_num(0.0), D.BF16 * D.slope(gd, activation).nan_to_num(0.0).abs() + 2.0 ** -20 * (1 + gd.abs().clamp_max(40))))


def test_training_step_on_a_side_stream_and_in_a_graph(cuda_device):
    """gated forward -> down projection -> its gradients -> the block's: eager, side stream, captured and replayed."""
    m, f, h = 200, 264, 136
    x, wg, wu = _block(cuda_device, m, f, h)
    wd, dy = _randn(cuda_device, h, f, 5, f ** -0.5), _randn(cuda_device, m, h, 6, 0.1)

    def step():
        hid, gate, up = ave.gemm_gated_transposed_b(x, wg, wu, save=True)
        y = gemm_pipeline_transposed_b(hid, wd)
        dh, dwd = ave.gemm_transposed_b_backward(dy, hid, wd)
        return (y, dwd, *ave.gemm_gated_backward(dh, x, wg, wu, gate, up))

    first = step()
    # against 64 bits without any inner rounding: each result goes through at most five roundings of 2^-8 / sqrt 3 in the mean
    # square (gate and up, the hidden state, its gradient, the inner gradients, the result)
    xd, gd_, ud_, wdd = (t.double().requires_grad_() for t in (x, wg, wu, wd))
    y = (D.act(xd @ gd_.T, "silu") * (xd @ ud_.T)) @ wdd.T
    grads = torch.autograd.grad(y, (wdd, xd, gd_, ud_), dy.double())
    for got, want in zip(first, (y.detach(), *grads)):
        assert (got.double() - want).norm() <= 5 * 2.0 ** -8 / 3 ** 0.5 * want.norm()
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    x.copy_(_randn(cuda_device, m, h, 11))
    wg.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(captured, step()))
    ave.check_device_status(cuda_device)


@pytest.mark.parametrize("m,n,k", [(40, 8200, 64), (8200, 40, 64), (9, 4096, 16), (300, 16392, 72), (8200, 264, 136), (130, 5000, 200)])
def test_long_sums_of_few_tiles(cuda_device, m, n, k):
    """Products of a few tiles and long sums: K is cut into ranges whose sums are added by a kernel of their own."""
    a, b, dout = _randn(cuda_device, m, k, 1), _randn(cuda_device, n, k, 2, k ** -0.5), _randn(cuda_device, m, n, 3, 0.1)
    got = ave.gemm_transposed_b_backward(dout, a, b)
    for g, w, what in zip(got, D.product_backward(dout, a, b), ("da", "db")):
        D.check(g, w, what)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(got, ave.gemm_transposed_b_backward(dout, a, b)))
    f, h = n, k
    wg, wu = _randn(cuda_device, f, h, 5, h ** -0.5), _randn(cuda_device, f, h, 6, h ** -0.5)
    gate, up = _randn(cuda_device, m, f, 7), _randn(cuda_device, m, f, 8)
    for g, w, what in zip(ave.gemm_gated_backward(dout, a, wg, wu, gate, up), D.gated_backward(dout, a, wg, wu, gate, up, "silu"), ("dx", "dw_gate", "dw_up")):
        D.check(g, w, what)
    ave.check_device_status(cuda_device)


def test_kept_products_feed_the_backward_pass_for_few_rows(cuda_device):
    """save=True on the streaming kernel (up to 16 rows) and on either side of its rule for large weights."""
    for m, f, h in ((1, 520, 264), (8, 8200, 1032), (9, 8200, 1032), (16, 4104, 2056), (12, 16, 8)):
        x, wg, wu = _block(cuda_device, m, f, h)
        kept = ave.gemm_gated_transposed_b(x, wg, wu, activation="gelu", save=True)
        for got, w, what in zip(kept, D.gated(x, wg, wu, "gelu"), ("out", "gate", "up")):
            D.check(got, w, f"{m}x{f}x{h} {what}")
        dout = _randn(cuda_device, m, f, 4, 0.1)
        for g, w in zip(ave.gemm_gated_backward(dout, x, wg, wu, *kept[1:], activation="gelu"),
                        D.gated_backward(dout, x, wg, wu, *kept[1:], "gelu")):
            D.check(g, w, f"{m}x{f}x{h}")
    ave.check_device_status(cuda_device)


def test_backward_captured_twice_and_replayed_at_once(cuda_device):
    """Two captured backward passes on streams of their own at the same time, next to eager calls: each has its own workspace."""
    m, f, h = 150, 1032, 264
    x, wg, wu = _block(cuda_device, m, f, h)
    gate, up = _randn(cuda_device, m, f, 5), _randn(cuda_device, m, f, 6)
    douts = [_randn(cuda_device, m, f, s, 0.1) for s in (7, 8, 9)]
    want = [ave.gemm_gated_backward(d, x, wg, wu, gate, up) for d in douts]
    graphs, got = [], []
    for d in douts[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(ave.gemm_gated_backward(d, x, wg, wu, gate, up))
        graphs.append(g)
    streams = [torch.cuda.Stream(cuda_device) for _ in range(3)]
    torch.cuda.synchronize()
    eager = []
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            eager.append(ave.gemm_gated_backward(douts[2], x, wg, wu, gate, up))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(p, q) for p, q in zip(got[i], want[i]))
    for e in eager:
        assert all(torch.equal(p, q) for p, q in zip(e, want[2]))
    ave.check_device_status(cuda_device)


def test_first_call_of_each_operator_inside_a_capture(cuda_device):
    """A fresh process: after the library's set-up, every operator's first call ever is a captured one."""
    import os
    import subprocess
    import sys

    code = """
import torch, avelang_b200 as ave
from avelang_b200 import _lib
_lib.ensure_init(0)
bf = torch.bfloat16
x, w = torch.randn(40, 64, device="cuda").to(bf), torch.randn(72, 64, device="cuda").to(bf)
def everything():
    q, v = ave.quantize_int8(x), ave.quantize_int8(w)
    out, gate, up = ave.gemm_gated_transposed_b(x, w, w, save=True)
    return (q.values, ave.gemm_int8_transposed_b(q, v), ave.gemm_int8_gated_transposed_b(q, v, v), out, gate, up,
            *ave.gemm_gated_backward(out, x, w, w, gate, up), *ave.gemm_transposed_b_backward(out, x, w))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = everything()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, everything()))
ave.check_device_status()
print("fine")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "fine" in run.stdout, run.stdout + run.stderr


@pytest.mark.parametrize("m,f,h", [(28, 1016, 6712), (40, 64, 8200), (300, 264, 4104), (17, 2056, 5008), (129, 520, 2048)])
def test_forward_with_long_sums(cuda_device, m, f, h):
    x, wg, wu = _block(cuda_device, m, f, h)
    for activation in ACTS:
        kept = ave.gemm_gated_transposed_b(x, wg, wu, activation=activation, save=True)
        for got, w, what in zip(kept, D.gated(x, wg, wu, activation), ("out", "gate", "up")):
            D.check(got, w, f"{activation} {what}")
        assert torch.equal(kept[0], ave.gemm_gated_transposed_b(x, wg, wu, activation=activation))
    ave.check_device_status(cuda_device)


@pytest.mark.parametrize("m", [2, 20, 200])
@pytest.mark.parametrize("activation", ACTS)
def test_far_arguments_forward(cuda_device, m, activation):
    """Gates over the whole range of bf16, through the streaming and the tile kernel: x is one-hot, so the gate is the weight itself."""
    g = torch.cat([torch.linspace(-40, 40, 1001), torch.tensor([1e4, -1e4, 1e18, -1e18, 3e38, -3e38, 1e-30])]).to(torch.bfloat16)
    f = g.numel() // 8 * 8
    wg, wu = (torch.zeros((f, 16), dtype=torch.bfloat16, device=cuda_device) for _ in range(2))
    wg[:, 3] = g[-f:].to(cuda_device)
    wu[:, 3] = 1.0
    x = torch.zeros((m, 16), dtype=torch.bfloat16, device=cuda_device)
    x[:, 3] = 1.0
    gd = wg[:, 3].double().expand(m, f)
    want = D.act(gd, activation)
    if activation == "gelu_tanh":
        want = torch.where(gd > 1e10, gd, torch.where(gd < -1e10, torch.zeros_like(gd), want))      # the cube overflows in the plain form
    got = ave.gemm_gated_transposed_b(x, wg, wu, activation=activation)
    D.check(got, (want, D.BF16 * want.abs() + 1e-37))


def test_gradients_beyond_two_to_the_31_elements(cuda_device):
    m, f, h = 66000, 32776, 8
    g = torch.Generator(device=cuda_device).manual_seed(0)
    dout, gate, up = (torch.randn((m, f), generator=g, device=cuda_device, dtype=torch.bfloat16) for _ in range(3))
    x, wg, wu = _randn(cuda_device, m, h, 4), _randn(cuda_device, f, h, 5), _randn(cuda_device, f, h, 6)
    dx, dwg, dwu = ave.gemm_gated_backward(dout, x, wg, wu, gate, up)
    ave.check_device_status(cuda_device)
    for rows in (slice(0, 2), slice(32767, 32770), slice(65534, 65538), slice(m - 2, m)):
        want = D.gated_backward(dout[rows], x[rows], wg, wu, gate[rows], up[rows], "silu")
        D.check(dx[rows], want[0], f"{rows}")
    for cols in (slice(0, 8), slice(16384, 16392), slice(f - 8, f)):
        want = D.gated_backward(dout[:, cols], x, wg[cols], wu[cols], gate[:, cols], up[:, cols], "silu")
        D.check(dwg[cols], want[1], f"{cols}")
        D.check(dwu[cols], want[2], f"{cols}")


@pytest.mark.parametrize("m,n,k", [(64, 72, 4104), (777, 1032, 4104), (300, 5000, 136), (2000, 264, 520)])
def test_operands_overwritten_right_after_a_call(cuda_device, m, n, k):
    """The second product of a backward pass starts before the first has ended: whatever is queued next still finds both done."""
    a, b, dout = _randn(cuda_device, m, k, 1), _randn(cuda_device, n, k, 2), _randn(cuda_device, m, n, 3)
    wg, wu, gate, up = b.clone(), b.clone(), _randn(cuda_device, m, n, 4), _randn(cuda_device, m, n, 5)
    da, db = ave.gemm_transposed_b_backward(dout, a, b)
    dx, dwg, dwu = ave.gemm_gated_backward(dout, a, wg, wu, gate, up)
    got = []
    for _ in range(20):
        got.append(ave.gemm_transposed_b_backward(dout, a, b))
        a.neg_()
        b.neg_()
        got.append(ave.gemm_gated_backward(dout, a, wg, wu, gate, up))
        dout.neg_()
        wg.neg_()
        wu.neg_()
    for i in range(20):
        # before iteration i all five have changed sign i times, and x once more before its second call
        assert torch.equal(got[2 * i][0], da) and torch.equal(got[2 * i][1], db)      # two changed signs each
        assert torch.equal(got[2 * i + 1][0], dx)                                    # dout and the weights
        assert torch.equal(got[2 * i + 1][1], -dwg) and torch.equal(got[2 * i + 1][2], -dwu)      # dout and x
    ave.check_device_status(cuda_device)


@pytest.mark.parametrize("m,n,k", [(8, 2552, 2048), (16, 120, 40008), (300, 128, 40008), (264, 2216, 2784), (777, 1032, 4104),
                                   (753, 2912, 288), (744, 7384, 248), (880, 1800, 160), (393, 3104, 448), (1024, 4096, 1024),
                                   (64, 4096, 4096), (1, 2048, 4104), (128, 8200, 1032)])
def test_second_product_ahead_of_the_first_ones_end(cuda_device, m, n, k):
    # the first product's last wave leaves SMs to the second's first clusters, in all four mixes of pairs and single CTAs
    a, b, dout = _randn(cuda_device, m, k, 1), _randn(cuda_device, n, k, 2, k ** -0.5), _randn(cuda_device, m, n, 3, 0.1)
    want = D.product_backward(dout, a, b)
    da = ave.gemm_transposed_b_backward(dout, a, b, need_db=False)[0]
    db = ave.gemm_transposed_b_backward(dout, a, b, need_da=False)[1]
    for _ in range(3):
        got = ave.gemm_transposed_b_backward(dout, a, b)
        for g, w, alone, what in zip(got, want, (da, db), ("da", "db")):
            D.check(g, w, what)
            assert torch.equal(g, alone)
    ave.check_device_status(cuda_device)


@pytest.mark.parametrize("m,f,h", [(8, 2824, 1664), (16, 1664, 1704), (32, 2672, 2736), (520, 1200, 2000), (1003, 2744, 1048), (424, 1488, 528),
                                   (1144, 1040, 216), (8, 80, 120), (1760, 1376, 488), (24, 5432, 2632), (1, 8200, 520), (128, 4096, 2048)])
def test_second_product_ahead_gated(cuda_device, m, f, h):
    x, wg, wu = _randn(cuda_device, m, h, 1), _randn(cuda_device, f, h, 2, h ** -0.5), _randn(cuda_device, f, h, 3, h ** -0.5)
    dout, gate, up = (_randn(cuda_device, m, f, s) for s in (4, 5, 6))
    got = ave.gemm_gated_backward(dout, x, wg, wu, gate, up)
    for g, w, what in zip(got, D.gated_backward(dout, x, wg, wu, gate, up, "silu"), ("dx", "dw_gate", "dw_up")):
        D.check(g, w, what)
    assert torch.equal(got[0], ave.gemm_gated_backward(dout, x, wg, wu, gate, up, need_dw=False)[0])
    alone = ave.gemm_gated_backward(dout, x, wg, wu, gate, up, need_dx=False)
    assert torch.equal(got[1], alone[1]) and torch.equal(got[2], alone[2])
    ave.check_device_status(cuda_device)
