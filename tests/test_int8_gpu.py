"""GPU tier: rows to 8-bit integers, integer products and the gated integer product, against 64-bit plain forms."""
import pytest
import torch

import avelang_b200 as ave
import dense_oracle as D

pytestmark = pytest.mark.gpu

ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def _randn(dev, rows, cols, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn((rows, cols), generator=g, device=dev) * scale).to(torch.bfloat16)


def _ints(dev, rows, k, seed, scale=0.02):
    g = torch.Generator(device=dev).manual_seed(seed)
    values = torch.randint(-127, 128, (rows, k), generator=g, device=dev, dtype=torch.int8)
    return ave.Int8Operand(values, torch.rand((rows,), generator=g, device=dev) * scale / k ** 0.5 + 1e-4)


# ------------------------------------------------------------------ quantise
@pytest.mark.parametrize("rows,k", [(1, 16), (9, 16), (3, 240), (17, 256), (5, 272), (2, 512), (8, 1024), (7, 1040), (3, 2048),
                                    (2, 2064), (5, 4096), (3, 4112), (301, 8192), (2, 8208), (2, 16384), (3, 16400), (2, 40000)])
def test_quantize_is_exact(cuda_device, rows, k):
    x = _randn(cuda_device, rows, k, k + rows) * torch.logspace(-20, 20, rows, device=cuda_device)[:, None].to(torch.bfloat16)
    q = ave.quantize_int8(x)
    values, scales = D.quantize_int8(x)
    assert torch.equal(q.values, values)
    # one fp32 division of an exact quotient
    assert torch.equal(q.scales, scales.float())


def test_quantize_every_pair_of_mantissas(cuda_device):
    """Every 8-bit significand as the row's maximum against every value down to 2^-10 of it: all ties and near-ties there are."""
    sig = torch.arange(128, 256, device=cuda_device, dtype=torch.float64)
    for exp in (-140, -126, -110, -8, 0, 100):
        top = (sig * 2.0 ** exp).to(torch.bfloat16)
        top = top[top > 0]
        below = torch.cat([(sig * 2.0 ** (exp - e)) for e in range(0, 11)])
        x = torch.minimum(below[None, :], top.double()[:, None])
        x = torch.cat([top.double()[:, None], x, -x], dim=1)
        x = torch.cat([x, torch.zeros((x.shape[0], (-x.shape[1]) % 16), device=cuda_device, dtype=torch.float64)], dim=1).to(torch.bfloat16)
        q = ave.quantize_int8(x)
        values, scales = D.quantize_int8(x)
        assert torch.equal(q.values, values), exp
        assert torch.equal(q.scales, scales.float()), exp


def test_quantize_special_rows(cuda_device):
    x = _randn(cuda_device, 8, 1088, 0)
    x[1] = 0.0
    x[2] = -0.0
    x[3, 77] = float("inf")
    x[4, 1087] = float("nan")
    x[5, 0] = float("-inf")
    x[6] = 3.3e38
    x[7] = 1e-40
    for k in (1088, 512):
        q = ave.quantize_int8(x[:, :k])
        finite = [0, 1, 2, 6, 7]
        values, scales = D.quantize_int8(x[finite, :k])
        assert torch.equal(q.values[finite], values) and torch.equal(q.scales[finite], scales.float())
        assert q.scales[1].item() == 1.0
        bad = [3, 5] + ([4] if k == 1088 else [])
        assert torch.isnan(q.scales[bad]).all() and not q.values[bad].any()
    w = _ints(cuda_device, 24, 1088, 3)
    y = ave.gemm_int8_transposed_b(ave.quantize_int8(x), w)
    assert torch.isnan(y[[3, 4, 5]]).all() and torch.isfinite(y[[0, 1, 2, 7]]).all()
    # row 6 is 3.3e38 throughout: its products are 3.3e38 times the sum of a weight row, past the range of bf16 (3.39e38) where that
    # sum is above 1.03, and then an infinity of the same sign
    ref, bound = D.int8_gemm(ave.quantize_int8(x[6:7]), w)
    over, within = ref.abs() > 3.42e38, ref.abs() < 3.36e38
    assert over.any() and within.any()
    assert torch.isinf(y[6:7][over]).all() and torch.equal(y[6:7][over].double().sign(), ref[over].sign())
    assert ((y[6:7].double() - ref).abs() <= bound)[within].all()


def test_quantize_strided_in_place(cuda_device):
    wide = _randn(cuda_device, 33, 200, 5)
    x = wide[:, 8:152]
    hold = torch.full((35, 192), 99, dtype=torch.int8, device=cuda_device)
    scales = torch.full((36,), -1.0, device=cuda_device)
    out = ave.Int8Operand(hold[1:34, 16:160], scales[:33])
    assert ave.quantize_int8(x, out=out) is out
    values, want = D.quantize_int8(x)
    assert torch.equal(out.values, values) and torch.equal(out.scales, want.float())
    hold[1:34, 16:160] = 99
    assert (hold == 99).all() and (scales[33:] == -1).all()
    assert ave.quantize_int8(x[:0]).shape == (0, 144)


# ------------------------------------------------------------------- product
SHAPES = [(1, 8, 16), (1, 4096, 1024), (3, 24, 48), (8, 136, 4112), (9, 2400, 80), (16, 9480, 272), (17, 8, 16), (33, 1000, 144),
          (128, 272, 1040), (129, 264, 128), (200, 2312, 400), (256, 512, 512), (300, 1336, 2064), (513, 4104, 1200), (1000, 760, 16)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_int8_gemm(cuda_device, m, n, k):
    a, b = _ints(cuda_device, m, k, 1), _ints(cuda_device, n, k, 2)
    bias = _randn(cuda_device, 1, n, 3)[0]
    for activation in ACTS:
        for bi in (None, bias):
            got = ave.gemm_int8_transposed_b(a, b, bias=bi, activation=activation)
            D.check(got, D.int8_gemm(a, b, bi, activation), f"{m}x{n}x{k} {activation} bias {bi is not None}")
    ave.check_device_status(cuda_device)


@pytest.mark.parametrize("m", [2, 16, 40, 130])
def test_int8_sums_are_exact(cuda_device, m):
    """Scales of 1 and sums below 2^24: the one rounding left is the one to bf16."""
    a, b = _ints(cuda_device, m, 512, 1), _ints(cuda_device, 264, 512, 2)
    a.scales.fill_(1.0)
    b.scales.fill_(1.0)
    want = (a.values.double() @ b.values.double().T).float().to(torch.bfloat16)
    assert torch.equal(ave.gemm_int8_transposed_b(a, b), want)


@pytest.mark.parametrize("m,n,k", [(40, 64, 8208), (890, 264, 8208), (12, 2504, 4112)])
def test_int8_sums_are_exact_when_cut(cuda_device, m, n, k):
    a, b = _ints(cuda_device, m, k, 1), _ints(cuda_device, n, k, 2)
    a.scales.fill_(1.0)
    b.scales.fill_(1.0)
    want = a.values.double() @ b.values.double().T
    assert want.abs().max() < 2 ** 24
    assert torch.equal(ave.gemm_int8_transposed_b(a, b), want.float().to(torch.bfloat16))


@pytest.mark.parametrize("m", [4, 24, 150])
@pytest.mark.parametrize("low", [-127, -128])
def test_int8_largest_sums(cuda_device, m, low):
    k = 131056
    a = ave.Int8Operand(torch.full((m, k), low, dtype=torch.int8, device=cuda_device), torch.ones(m, device=cuda_device))
    b = ave.Int8Operand(torch.full((16, k), low, dtype=torch.int8, device=cuda_device), torch.ones(16, device=cuda_device))
    b.values[8:] = 127
    got = ave.gemm_int8_transposed_b(a, b)
    want = (a.values.double() @ b.values.double().T).float().to(torch.bfloat16)
    assert torch.equal(got, want)


@pytest.mark.parametrize("m", [5, 70, 270])
def test_int8_strides_and_out(cuda_device, m):
    av = torch.randint(-127, 128, (m, 400), device=cuda_device, dtype=torch.int8)
    bv = torch.randint(-127, 128, (104, 352), device=cuda_device, dtype=torch.int8)
    a = ave.Int8Operand(av[:, 16:320], torch.rand(m, device=cuda_device))
    b = ave.Int8Operand(bv[:, 32:336], torch.rand(104, device=cuda_device))
    hold = torch.full((m + 2, 160), 7.0, dtype=torch.bfloat16, device=cuda_device)
    out = hold[1:m + 1, 24:128]
    assert ave.gemm_int8_transposed_b(a, b, out=out, activation="silu") is out
    D.check(out, D.int8_gemm(a, b, None, "silu"))
    out.fill_(7.0)
    assert (hold == 7.0).all()
    wu = ave.Int8Operand(bv[:, 0:304], torch.rand(104, device=cuda_device))
    assert ave.gemm_int8_gated_transposed_b(a, b, wu, out=out) is out
    D.check(out, D.int8_gated(a, b, wu, "silu"))
    out.fill_(7.0)
    assert (hold == 7.0).all()


@pytest.mark.parametrize("m,f,k", [(1, 8, 16), (1, 4104, 1024), (7, 136, 208), (16, 24, 4112), (17, 8, 16), (64, 1000, 144), (128, 520, 272),
                                   (129, 264, 128), (300, 1336, 1040), (513, 2056, 400)])
def test_int8_gated(cuda_device, m, f, k):
    a, wg, wu = _ints(cuda_device, m, k, 1), _ints(cuda_device, f, k, 2), _ints(cuda_device, f, k, 3)
    for activation in ACTS:
        got = ave.gemm_int8_gated_transposed_b(a, wg, wu, activation=activation)
        D.check(got, D.int8_gated(a, wg, wu, activation), f"{m}x{f}x{k} {activation}")
    ave.check_device_status(cuda_device)


def test_empty_products(cuda_device):
    a, b = _ints(cuda_device, 5, 64, 1), _ints(cuda_device, 24, 64, 2)
    none = ave.Int8Operand(a.values[:0], a.scales[:0])
    assert ave.gemm_int8_transposed_b(none, b).shape == (0, 24)
    assert ave.gemm_int8_transposed_b(a, none).shape == (5, 0)
    assert ave.gemm_int8_gated_transposed_b(none, b, b).shape == (0, 24)
    assert ave.gemm_int8_gated_transposed_b(a, none, none).shape == (5, 0)


@pytest.mark.parametrize("m", [1, 16, 50, 400])
def test_serving_block_on_a_side_stream_and_in_graphs(cuda_device, m):
    """quantise -> gated product -> quantise -> product: eager, on a side stream, and captured twice and replayed with other inputs."""
    h, f = 272, 528
    wg, wu = ave.quantize_int8(_randn(cuda_device, f, h, 1, 0.1)), ave.quantize_int8(_randn(cuda_device, f, h, 2, 0.1))
    wd = ave.quantize_int8(_randn(cuda_device, h, f, 3, 0.1))

    def block(x):
        mid = ave.gemm_int8_gated_transposed_b(ave.quantize_int8(x), wg, wu)
        return mid, ave.gemm_int8_transposed_b(ave.quantize_int8(mid), wd)

    x = _randn(cuda_device, m, h, 4)
    mid, y = block(x)
    D.check(mid, D.int8_gated(ave.Int8Operand(*D.quantize_int8(x)), wg, wu, "silu"))
    D.check(y, D.int8_gemm(ave.Int8Operand(*D.quantize_int8(mid)), wd))
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        mid2, y2 = block(x)
    side.synchronize()
    assert torch.equal(mid, mid2) and torch.equal(y, y2)
    inputs, graphs, results = [x.clone(), x.clone()], [], []
    for xi in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(block(xi))
        graphs.append(graph)
    for i, seed in ((0, 7), (1, 8), (0, 9)):
        inputs[i].copy_(_randn(cuda_device, m, h, seed))
        graphs[i].replay()
        torch.cuda.synchronize()
        want = block(inputs[i])
        assert torch.equal(results[i][0], want[0]) and torch.equal(results[i][1], want[1])
    # both at once, on streams of their own
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            for _ in range(5):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        want = block(inputs[i])
        assert torch.equal(results[i][1], want[1])
    ave.check_device_status(cuda_device)


def test_both_sides_of_the_streaming_rule(cuda_device):
    """Few rows go to the streaming kernel or to the tile kernel by the number of weight rows and the length of K."""
    for n, k in ((2360, 4112), (2400, 4112), (4728, 272), (4760, 272), (4760, 8192), (4760, 8208)):
        b = _ints(cuda_device, n, k, 2)
        for m in (1, 8, 9, 16):
            a = _ints(cuda_device, m, k, m)
            D.check(ave.gemm_int8_transposed_b(a, b, activation="silu"), D.int8_gemm(a, b, None, "silu"), f"{m}x{n}x{k}")
    for f in (1176, 1192, 2392):
        wg, wu = _ints(cuda_device, f, 4112, 5), _ints(cuda_device, f, 4112, 6)
        for m in (3, 9, 13, 16):
            a = _ints(cuda_device, m, 4112, m)
            D.check(ave.gemm_int8_gated_transposed_b(a, wg, wu), D.int8_gated(a, wg, wu, "silu"), f"gated {m}x{f}")
    ave.check_device_status(cuda_device)


@pytest.mark.parametrize("m,n,k", [(40, 64, 16384), (17, 3000, 8208), (300, 264, 12304), (890, 512, 11120), (130, 1032, 4096), (9, 2504, 16400)])
def test_long_sums_of_few_tiles(cuda_device, m, n, k):
    """K cut into ranges: the integer sums stay exact, whatever the cut."""
    a, b, c = _ints(cuda_device, m, k, 1), _ints(cuda_device, n, k, 2), _ints(cuda_device, n, k, 3)
    bias = _randn(cuda_device, 1, n, 3)[0]
    for activation in ACTS:
        D.check(ave.gemm_int8_transposed_b(a, b, bias=bias, activation=activation), D.int8_gemm(a, b, bias, activation), f"{activation}")
        D.check(ave.gemm_int8_gated_transposed_b(a, b, c, activation=activation), D.int8_gated(a, b, c, activation), f"gated {activation}")
    hold = torch.full((m + 2, n + 32), 7.0, dtype=torch.bfloat16, device=cuda_device)
    out = hold[1:m + 1, 16:n + 16]
    ave.gemm_int8_transposed_b(a, b, out=out)
    assert torch.equal(out, ave.gemm_int8_transposed_b(a, b))
    out.fill_(7.0)
    assert (hold == 7.0).all()
    ave.check_device_status(cuda_device)


def test_results_beyond_two_to_the_31_elements(cuda_device):
    m, n, k = 66000, 32776, 32
    a, b = _ints(cuda_device, m, k, 1), _ints(cuda_device, n, k, 2)
    got = ave.gemm_int8_transposed_b(a, b)
    for rows in (slice(0, 3), slice(32767, 32771), slice(65530, 65540), slice(m - 3, m)):
        part = ave.Int8Operand(a.values[rows], a.scales[rows].clone())
        D.check(got[rows], D.int8_gemm(part, b), f"{rows}")
    x = got[:, :16384]      # 1.08e9 elements at a row stride of 32776
    q = ave.quantize_int8(x)
    for rows in (slice(0, 2), slice(65533, 65540), slice(m - 2, m)):
        values, scales = D.quantize_int8(x[rows])
        assert torch.equal(q.values[rows], values) and torch.equal(q.scales[rows], scales.float())
    ave.check_device_status(cuda_device)


def test_two_host_threads_on_streams_of_their_own(cuda_device):
    import threading

    shapes = [(1, 1000, 1024), (40, 520, 272), (300, 264, 528), (16, 4104, 1040)]
    cases = [(_ints(cuda_device, m, k, 1), _ints(cuda_device, n, k, 2)) for m, n, k in shapes]
    want = [ave.gemm_int8_transposed_b(a, b, activation="gelu") for a, b in cases]
    torch.cuda.synchronize()
    bad = []

    def work(seed):
        stream = torch.cuda.Stream(cuda_device)
        with torch.cuda.stream(stream):
            for i in range(100):
                j = (i * seed) % len(cases)
                if not torch.equal(ave.gemm_int8_transposed_b(*cases[j], activation="gelu"), want[j]):
                    bad.append((seed, i))

    threads = [threading.Thread(target=work, args=(s,)) for s in (1, 3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    ave.check_device_status(cuda_device)


@pytest.mark.parametrize("m", [3, 30, 300])
@pytest.mark.parametrize("activation", ACTS)
def test_far_arguments(cuda_device, m, activation):
    """Arguments of the activation over a wide range, from the scales: codes of 1 and -1, scales up to 1e30."""
    n = 1008
    a = ave.Int8Operand(torch.zeros((m, 32), dtype=torch.int8, device=cuda_device), torch.ones(m, device=cuda_device))
    a.values[:, 5] = 1
    b = ave.Int8Operand(torch.zeros((n, 32), dtype=torch.int8, device=cuda_device), torch.logspace(-20, 30, n, device=cuda_device))
    b.values[::2, 5] = 1
    b.values[1::2, 5] = -1
    want, bound = D.int8_gemm(a, b, None, activation)
    if activation == "gelu_tanh":
        z = a.values[:, 5:6].double() * b.values[:, 5].double() * b.scales.double()
        want = torch.where(z > 1e10, z, torch.where(z < -1e10, torch.zeros_like(z), want))      # the cube overflows in the plain form
        bound = D.BF16 * want.abs() + 1.13 * 4 * 2.0 ** -24 * z.abs()
    D.check(ave.gemm_int8_transposed_b(a, b, activation=activation), (want, bound))


@pytest.mark.parametrize("m", [1, 12, 60, 300])
def test_one_operand_overwritten_again_and_again(cuda_device, m):
    """Each kernel is launched under the previous one's tail: the product sees the codes and scales of its own step."""
    k, n = 1040, 520
    xs = [_randn(cuda_device, m, k, s, 10.0 ** (s % 7 - 3)) for s in range(14)]
    w = _ints(cuda_device, n, k, 99)
    want = [ave.gemm_int8_transposed_b(ave.quantize_int8(x), w) for x in xs]
    torch.cuda.synchronize()
    q = ave.quantize_int8(xs[0])
    for _ in range(10):
        got = [ave.gemm_int8_transposed_b(ave.quantize_int8(x, out=q), w) for x in xs]
        for g, e in zip(got, want):
            assert torch.equal(g, e)


@pytest.mark.parametrize("m,n,k", [(20, 520, 128), (130, 1000, 64), (300, 2056, 272), (257, 4096, 1024)])
def test_results_on_and_off_32_bytes(cuda_device, m, n, k):
    # rows that lie on 32 bytes are stored in another way than rows on 16: same bits, and nothing beside them is touched
    a, b, bias = _ints(cuda_device, m, k, 1, 1.0), _ints(cuda_device, n, k, 2, 1.0), _randn(cuda_device, 1, n, 3)[0]
    want = ave.gemm_int8_transposed_b(a, b, bias=bias, activation="gelu")
    wide = (n + 15) // 16 * 16
    for width, first in ((wide + 32, 16), (wide + 32, 8), (wide + 40, 16), (wide + 40, 24)):
        hold = torch.full((m + 2, width), 7.0, dtype=torch.bfloat16, device=cuda_device)
        out = hold[1:m + 1, first:first + n]
        assert ave.gemm_int8_transposed_b(a, b, out=out, bias=bias, activation="gelu") is out
        assert torch.equal(out, want)
        out.fill_(7.0)
        assert (hold == 7.0).all()
    ave.check_device_status(cuda_device)
