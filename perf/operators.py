"""Cases, inputs and plain forms of the integer products, the gated feed-forward block and the products' gradients.

The operators: rows quantised to 8-bit integers, the product of two such operands with a scale for each token and each
channel, the same with two weights joined by an activation, the gated block ``act(x Wg^T) * (x Wu^T)`` on bf16 with its
backward pass, and the backward pass of the bf16 product ``A B^T``.
"""
import math

import torch

own = False

ACTIVATIONS = ("silu", "gelu", "gelu_tanh", "relu", "none")


def listed():
    return [
        # one token's activations on their way into an integer product: all latency
        dict(name="quantize_1x4096", op="quantize", m=1, k=4096, wide=False),
        # a whole prompt's activations
        dict(name="quantize_8192x8192", op="quantize", m=8192, k=8192, wide=False),
        # decode of a batch of 16 through one projection: the weights are read once
        dict(name="int8_16x28672x8192", op="int8", m=16, n=28672, k=8192, act="none", bias=False),
        # a prompt of 8192 tokens through a square layer with bias and activation
        dict(name="int8_8192x8192x8192", op="int8", m=8192, n=8192, k=8192, act="gelu_tanh", bias=True),
        # one token through the gated half of a feed-forward block
        dict(name="int8_gated_1x28672x8192", op="int8_gated", m=1, f=28672, k=8192, act="silu"),
        # a prompt through it
        dict(name="int8_gated_4096x28672x8192", op="int8_gated", m=4096, f=28672, k=8192, act="silu"),
        # the block in bf16 for one token
        dict(name="gated_1x8192x4096", op="gated", m=1, f=8192, h=4096, act="silu", save=False, wide=False),
        # a training step's forward pass, which keeps both projections for the backward pass
        dict(name="gated_save_4096x16384x4096", op="gated", m=4096, f=16384, h=4096, act="silu", save=True, wide=False),
        # the backward pass of a small block on a batch of no round size
        dict(name="gated_backward_1003x2744x1048", op="gated_backward", m=1003, f=2744, h=1048, act="gelu_tanh", wide=False),
        # a training step's backward pass
        dict(name="gated_backward_8192x16384x4096", op="gated_backward", m=8192, f=16384, h=4096, act="silu", wide=False),
        # gradients of one product, no round sizes
        dict(name="product_backward_777x1032x4104", op="product_backward", m=777, n=1032, k=4104),
        # gradients of the down projection's product in a training step
        dict(name="product_backward_8192x4096x16384", op="product_backward", m=8192, n=4096, k=16384),
    ]


def _spread(rng, low, high, multiple=1):
    """A size between low and high, even over its logarithm, a multiple of `multiple`."""
    v = math.exp(rng.uniform(math.log(low), math.log(high + 1)))
    return max(low, min(high, int(v) // multiple * multiple))


def draw(rng):
    op = rng.choice(("quantize", "int8", "int8", "int8_gated", "gated", "gated", "gated_backward", "gated_backward", "product_backward"))
    case = dict(op=op, m=_spread(rng, 1, 8192))
    if op == "quantize":
        case |= dict(k=_spread(rng, 64, 16384, 16), wide=rng.random() < 0.3)
    elif op == "int8":
        case |= dict(n=_spread(rng, 64, 28672, 8), k=_spread(rng, 64, 16384, 16), act=rng.choice(ACTIVATIONS), bias=rng.random() < 0.5)
    elif op == "int8_gated":
        case |= dict(f=_spread(rng, 64, 28672, 8), k=_spread(rng, 64, 8192, 16), act=rng.choice(ACTIVATIONS))
    elif op == "gated":
        case |= dict(f=_spread(rng, 64, 28672, 8), h=_spread(rng, 64, 8192, 8), act=rng.choice(ACTIVATIONS), save=rng.random() < 0.5,
                     wide=rng.random() < 0.3)
    elif op == "gated_backward":
        case |= dict(f=_spread(rng, 64, 16384, 8), h=_spread(rng, 64, 8192, 8), act=rng.choice(ACTIVATIONS), wide=rng.random() < 0.3)
    else:
        case |= dict(n=_spread(rng, 64, 16384, 8), k=_spread(rng, 64, 16384, 8))
    most = max(work(c)["flops"] for c in listed())
    while work(case)["flops"] > most:
        case["m"] = (case["m"] + 1) // 2
    return case


def work(case):
    op, m = case["op"], case["m"]
    if op == "quantize":
        k = case["k"]
        return {"bytes": m * k * 3 + m * 4, "flops": m * k * 4}
    if op == "int8":
        n, k = case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if op == "int8_gated":
        f, k = case["f"], case["k"]
        return {"bytes": m * k + 2 * f * k + 4 * (m + 2 * f) + 2 * m * f, "flops": 4 * m * f * k}
    if op == "gated":
        f, h = case["f"], case["h"]
        return {"bytes": 2 * (m * h + 2 * f * h + m * f * (3 if case["save"] else 1)), "flops": 4 * m * f * h}
    if op == "gated_backward":
        f, h = case["f"], case["h"]
        return {"bytes": 2 * (3 * m * f + 2 * m * h + 4 * f * h), "flops": 8 * m * f * h}
    n, k = case["n"], case["k"]
    return {"bytes": 2 * (m * n + 2 * m * k + 2 * n * k), "flops": 4 * m * n * k}


def _activations(g, rows, cols, wide=False):
    """Hidden states: normal, with a few channels of large values; `wide`: a column block of a wider matrix."""
    x = torch.randn((rows, cols + (64 if wide else 0)), generator=g, device="cuda")
    x[:, :: 997] *= 12.0
    return x.to(torch.bfloat16)[:, :cols]


def _weights(g, rows, cols):
    return (torch.randn((rows, cols), generator=g, device="cuda") * cols ** -0.5).to(torch.bfloat16)


def _integers(x):
    """Rows of x as 8-bit integers with a scale each."""
    x = x.float()
    most = x.abs().amax(dim=1, keepdim=True)
    most = torch.where(most > 0, most, torch.full_like(most, 127.0))
    return torch.round(x * 127.0 / most).to(torch.int8), (most / 127.0).reshape(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op, m = case["op"], case["m"]
    s = dict(case)
    if op == "quantize":
        s["x"] = _activations(g, m, case["k"], case["wide"])
    elif op in ("int8", "int8_gated"):
        k = case["k"]
        s["a"] = _integers(_activations(g, m, k))
        if op == "int8":
            s["b"] = _integers(_weights(g, case["n"], k))
            s["b_bias"] = (0.1 * torch.randn((case["n"],), generator=g, device="cuda")).to(torch.bfloat16) if case["bias"] else None
        else:
            s["gate"], s["up"] = _integers(_weights(g, case["f"], k)), _integers(_weights(g, case["f"], k))
    elif op in ("gated", "gated_backward"):
        f, h = case["f"], case["h"]
        s["x"] = _activations(g, m, h, case["wide"])
        s["w_gate"], s["w_up"] = _weights(g, f, h), _weights(g, f, h)
        if op == "gated_backward":
            s["gate"], s["up"] = s["x"] @ s["w_gate"].T, s["x"] @ s["w_up"].T      # what the forward pass kept
            s["dout"] = (0.01 * torch.randn((m, f), generator=g, device="cuda")).to(torch.bfloat16)
    else:
        n, k = case["n"], case["k"]
        s["a"], s["b"] = _activations(g, m, k), _weights(g, n, k)
        s["dout"] = (0.01 * torch.randn((m, n), generator=g, device="cuda")).to(torch.bfloat16)
    return s


def _act(x, act):
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * x * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (x + 0.044715 * x * x * x)))
    return torch.where(x > 0, x, torch.zeros_like(x)) if act == "relu" else x


def _act_slope(x, act):
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-x))
        return p * (1.0 + x * (1.0 - p))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(x * 0.5 ** 0.5)) + x * torch.exp(-0.5 * x * x) * (2.0 * math.pi) ** -0.5
    if act == "gelu_tanh":
        c = (2.0 / math.pi) ** 0.5
        t = torch.tanh(c * (x + 0.044715 * x * x * x))
        return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * x * x)
    return (x > 0).to(x.dtype) if act == "relu" else torch.ones_like(x)


def _run_own(s):
    import avelang_b200 as ave

    op = s["op"]
    if op == "quantize":
        q = ave.quantize_int8(s["x"])
        return {"values": q.values, "scales": q.scales}
    if op == "int8":
        return ave.gemm_int8_transposed_b(ave.Int8Operand(*s["a"]), ave.Int8Operand(*s["b"]), bias=s["b_bias"], activation=s["act"])
    if op == "int8_gated":
        return ave.gemm_int8_gated_transposed_b(ave.Int8Operand(*s["a"]), ave.Int8Operand(*s["gate"]), ave.Int8Operand(*s["up"]),
                                                activation=s["act"])
    if op == "gated":
        return ave.gemm_gated_transposed_b(s["x"], s["w_gate"], s["w_up"], activation=s["act"], save=s["save"])
    if op == "gated_backward":
        return ave.gemm_gated_backward(s["dout"], s["x"], s["w_gate"], s["w_up"], s["gate"], s["up"], activation=s["act"])
    return ave.gemm_transposed_b_backward(s["dout"], s["a"], s["b"])


def run(s):
    if own:
        return _run_own(s)
    op = s["op"]
    if op == "quantize":
        values, scales = _integers(s["x"])
        return {"values": values, "scales": scales}
    if op in ("int8", "int8_gated"):
        a, sa = s["a"][0].float(), s["a"][1][:, None]
        if op == "int8":
            b, sb = s["b"]
            y = (a @ b.float().T) * sa * sb
            return _act(y if s["b_bias"] is None else y + s["b_bias"].float(), s["act"]).to(torch.bfloat16)
        (wg, sg), (wu, su) = s["gate"], s["up"]
        return (_act((a @ wg.float().T) * sa * sg, s["act"]) * ((a @ wu.float().T) * sa * su)).to(torch.bfloat16)
    if op == "gated":
        x = s["x"].float()
        gate, up = x @ s["w_gate"].float().T, x @ s["w_up"].float().T
        out = (_act(gate, s["act"]) * up).to(torch.bfloat16)
        return (out, gate.to(torch.bfloat16), up.to(torch.bfloat16)) if s["save"] else out
    if op == "gated_backward":
        d, gate, x = s["dout"].float(), s["gate"].float(), s["x"].float()
        d_up = d * _act(gate, s["act"])
        d_gate = d * s["up"].float() * _act_slope(gate, s["act"])
        dx = d_gate @ s["w_gate"].float() + d_up @ s["w_up"].float()
        return dx.to(torch.bfloat16), (d_gate.T @ x).to(torch.bfloat16), (d_up.T @ x).to(torch.bfloat16)
    d = s["dout"].float()
    return (d @ s["b"].float()).to(torch.bfloat16), (d.T @ s["a"].float()).to(torch.bfloat16)


def exact(case, seed):
    s = prepare(case, seed)
    op, act = case["op"], case.get("act")
    wide = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    sigmoid = torch.special.expit

    def cdf(z):
        return 0.5 * torch.special.erfc(z * -math.sqrt(0.5))

    def cubic(z):      # twice the argument of the tanh form
        return math.sqrt(8.0 / math.pi) * (z + 0.044715 * z ** 3)

    value = {"silu": lambda z: z * sigmoid(z), "gelu": lambda z: z * cdf(z), "gelu_tanh": lambda z: z * sigmoid(cubic(z)),
             "relu": lambda z: z.clamp_min(0.0), "none": lambda z: z}.get(act)
    slope = {"silu": lambda z: sigmoid(z) + z * sigmoid(z) * sigmoid(-z),
             "gelu": lambda z: cdf(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi),
             "gelu_tanh": lambda z: sigmoid(cubic(z)) + z * sigmoid(cubic(z)) * sigmoid(-cubic(z)) * math.sqrt(8.0 / math.pi) * (1 + 0.134145 * z * z),
             "relu": lambda z: (z > 0).double(), "none": lambda z: torch.ones_like(z)}.get(act)
    if op == "quantize":
        x = wide["x"]
        top = x.abs().max(dim=1).values
        top = torch.where(top == 0, 127.0, top)
        return {"values": (x * 127 / top.unsqueeze(1)).round().to(torch.int8), "scales": top / 127}
    if op in ("int8", "int8_gated"):
        a = s["a"][0].double() * s["a"][1].double().unsqueeze(1)
        weight = lambda w: (w[0].double() * w[1].double().unsqueeze(1)).t()  # noqa: E731
        if op == "int8_gated":
            return value(torch.mm(a, weight(s["gate"]))) * torch.mm(a, weight(s["up"]))
        y = torch.mm(a, weight(s["b"]))
        return value(y + wide["b_bias"] if case["bias"] else y)
    if op == "gated":
        gate, up = torch.mm(wide["x"], wide["w_gate"].t()), torch.mm(wide["x"], wide["w_up"].t())
        return (value(gate) * up, gate, up) if case["save"] else value(gate) * up
    if op == "gated_backward":
        to_gate = wide["dout"] * wide["up"] * slope(wide["gate"])
        to_up = wide["dout"] * value(wide["gate"])
        both = torch.cat((to_gate, to_up), dim=1)
        dw = torch.mm(both.t(), wide["x"])
        return torch.mm(both, torch.cat((wide["w_gate"], wide["w_up"]))), dw[: case["f"]], dw[case["f"]:]
    return torch.mm(wide["dout"], wide["b"]), torch.mm(wide["dout"].t(), wide["a"])
