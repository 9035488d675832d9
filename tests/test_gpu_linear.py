"""GPU tests of esmm_linear and esmm_epilogue_backward against 64-bit products: operand layouts and types, every part of the
epilogue, ragged and smallest sizes, each of its kernels, streams, graphs, and a layer's gradients."""
import pytest
import torch

import dense_ops as d

pytestmark = pytest.mark.gpu


def operands(m, n, k, t, trans_a=False, trans_b=False, seed=0, std=1.0):
    """(A as stored, B as stored, op(A) and op(B) in 64 bits)"""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    a = torch.randn((m, k), generator=gen, device="cuda") * std
    b = torch.randn((k, n), generator=gen, device="cuda") / k ** 0.5
    a, b = a.to(d.TYPES[t]), b.to(d.TYPES[t])
    return (a.t().contiguous() if trans_a else a, b.t().contiguous() if trans_b else b, a.double(), b.double())


def check(pkg, m, n, k, t, out="", trans_a=False, trans_b=False, activation="none", bias=False, residual=False, pre=False, scales=False,
          seed=0, stream=0, inplace=False):
    out = out or t
    trans_b = trans_b or t == "e4m3"
    a, b, a64, b64 = operands(m, n, k, t, trans_a, trans_b, seed)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    ot = d.TYPES[out]
    bias_t = torch.randn((n,), generator=gen, device="cuda").to(ot) if bias else None
    res = torch.randn((m, n), generator=gen, device="cuda").to(ot) if residual else None
    sa = torch.rand((m,), generator=gen, device="cuda") + 0.5 if scales else None
    sb = torch.rand((n,), generator=gen, device="cuda") + 0.5 if scales else None
    c, c_ok = d.guarded(m, n, ot)
    p, p_ok = d.guarded(m, n, ot)
    c.fill_(float("nan"))
    if inplace:
        c.copy_(res)
    ptr = lambda x: 0 if x is None else x.data_ptr()  # noqa: E731
    pkg.linear(m, n, k, d.code(pkg, t), ptr(a), ptr(b), d.code(pkg, out), ptr(c), trans_a=int(trans_a), trans_b=int(trans_b), a_scale=ptr(sa),
               b_scale=ptr(sb), bias=ptr(bias_t), residual=ptr(c if inplace else res), pre=ptr(p) if pre else 0,
               activation=d.act_code(pkg, activation), stream=stream)
    pkg.device_status(stream)
    z, want, mag = d.linear(a64, b64, sa, sb, bias_t, activation, res)
    u = d.half_step(out)
    # an activation's slope is at most 1.13; its own arithmetic and the residual's addition are a few 32-bit roundings
    off = 1.13 * d.sum_error(mag, k) + 2.0 ** -20 * (z.abs() + want.abs())
    d.assert_close(c, want, off + u * (want.abs() + off) + d.smallest(out), "C")
    if pre:
        d.assert_close(p, z, d.sum_error(mag, k) + u * (z.abs() + d.sum_error(mag, k)) + d.smallest(out), "pre")
    assert c_ok() and p_ok()
    return c


SIZES = [(1, 8, 16), (1, 128, 64), (7, 200, 48), (16, 520, 1040), (33, 72, 256), (127, 136, 2000), (128, 128, 128), (129, 264, 80), (300, 392, 528),
         (513, 1032, 336)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("t", ["bf16", "f16", "e4m3"])
def test_sizes(cuda, pkg, t, m, n, k):
    check(pkg, m, n, k, t, out="bf16" if t == "e4m3" else t)
    check(pkg, m, n, k, t, out="f16" if t == "e4m3" else t, activation="silu", bias=True, residual=True, pre=True, scales=True, seed=3)


@pytest.mark.parametrize("pair", [0, 64, 128, 192, 256])
@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (40, 72, 72), (256, 256, 64), (264, 520, 200), (1000, 1512, 328)])
@pytest.mark.parametrize("trans", ["nn", "nt", "tn"])
def test_kernels_and_layouts(cuda, pkg, tuning, pair, m, n, k, trans):
    if trans == "tn":
        m = -(-m // 8) * 8
    tuning("LINEAR_PAIR", pair)
    for t in ("bf16", "f16"):
        check(pkg, m, n, k, t, trans_a=trans == "tn", trans_b=trans == "nt", activation="gelu", bias=True, residual=True, pre=True)


@pytest.mark.parametrize("pair", [0, 64, 128, 192, 256])
def test_e4m3_kernels(cuda, pkg, tuning, pair):
    tuning("LINEAR_PAIR", pair)
    for (m, n, k) in [(1, 8, 16), (264, 520, 400), (700, 776, 1168)]:
        check(pkg, m, n, k, "e4m3", out="bf16", activation="gelu_tanh", bias=True, residual=True, pre=True, scales=True)


@pytest.mark.parametrize("pair,tail", [(128, 64), (192, 64), (192, 128), (256, 64), (256, 128), (256, 192)])
def test_two_tile_widths(cuda, pkg, tuning, pair, tail):
    tuning("LINEAR_PAIR", pair)
    tuning("LINEAR_TAIL", tail)
    for trans in ("nn", "nt", "tn"):
        check(pkg, 520, 1512, 200, "bf16", trans_a=trans == "tn", trans_b=trans == "nt", activation="silu", bias=True, residual=True, pre=True)
    check(pkg, 300, 2056, 400, "e4m3", out="f16", bias=True, residual=True, scales=True)
    check(pkg, 9, pair + 8, 64, "f16", bias=True)


@pytest.mark.parametrize("pair", [288, 320, 352, 384, 480, 512])
@pytest.mark.parametrize("k", [200, 1088])
def test_tiles_wider_than_an_instruction(cuda, pkg, tuning, pair, k):
    """Two accumulators side by side, the last piece 32 or 64 columns wide; the last tile's columns end inside its first or second part."""
    tuning("LINEAR_PAIR", pair)
    for trans in ("nn", "nt", "tn"):
        for n in (pair, 3 * pair - 40, 2 * pair + 104):
            check(pkg, 520, n, k, "bf16", trans_a=trans == "tn", trans_b=trans == "nt", activation="silu", bias=True, residual=True, pre=True)
    check(pkg, 300, 2 * pair + 8, -(-k // 16) * 16, "e4m3", out="f16", bias=True, residual=True, scales=True, activation="gelu")
    check(pkg, 300, 2 * pair + 8, k, "f16", trans_b=True, bias=True, residual=True, inplace=True)
    check(pkg, 9, 8, k, "bf16", trans_b=True)


@pytest.mark.parametrize("split", [1, 2, 3, 8])
@pytest.mark.parametrize("columns", [64, 128])
def test_parts_of_k(cuda, pkg, tuning, split, columns):
    tuning("LINEAR_PAIR", 0)
    tuning("LINEAR_SPLIT", split)
    tuning("LINEAR_COLUMNS", columns)
    for t, (m, n, k) in [("bf16", (5, 136, 1000)), ("bf16", (200, 264, 72)), ("e4m3", (130, 72, 2064)), ("f16", (128, 320, 640))]:
        check(pkg, m, n, k, t, out="bf16" if t == "e4m3" else t, bias=True, residual=True, scales=True)


@pytest.mark.parametrize("split", [4, 5, 6, 7])
@pytest.mark.parametrize("columns", [64, 128])
def test_other_parts_of_k(cuda, pkg, tuning, split, columns):
    """The numbers of parts that the library chooses beside those above, and the odd ones that only the hook asks for; K steps that do not divide among them."""
    tuning("LINEAR_PAIR", 0)
    tuning("LINEAR_SPLIT", split)
    tuning("LINEAR_COLUMNS", columns)
    for t, (m, n, k) in [("bf16", (5, 136, 1000)), ("bf16", (200, 264, 72)), ("e4m3", (130, 72, 2064)), ("f16", (128, 320, 640)), ("bf16", (17, 128, 4160))]:
        check(pkg, m, n, k, t, out="bf16" if t == "e4m3" else t, bias=True, residual=True, scales=True, pre=True, activation="silu")
        check(pkg, m, n, k, t, out="bf16" if t == "e4m3" else t)


@pytest.mark.parametrize("activation", d.ACTS)
@pytest.mark.parametrize("pair", [0, 256])
def test_epilogue_parts(cuda, pkg, tuning, activation, pair):
    tuning("LINEAR_PAIR", pair)
    for bits in range(16):
        check(pkg, 130, 200, 96, "bf16", activation=activation, bias=bool(bits & 1), residual=bool(bits & 2), pre=bool(bits & 4), scales=bool(bits & 8),
              seed=bits)


@pytest.mark.parametrize("pair", [0, 64, 128, 192, 256])
def test_residual_in_place(cuda, pkg, tuning, pair):
    tuning("LINEAR_PAIR", pair)
    check(pkg, 300, 328, 128, "f16", bias=True, residual=True, inplace=True, activation="relu")


@pytest.mark.parametrize("pair", [64, 128, 192, 256])
@pytest.mark.parametrize("k", [64, 1088])
def test_many_tiles_per_cta(cuda, pkg, tuning, pair, k):
    """Short K (two staging boxes per warp) and long (one), one and two pieces per warp and tile, edges in the last tile row and column."""
    tuning("LINEAR_PAIR", pair)
    m, n = (2320, 2072) if pair < 256 else (2320, 4136)
    for residual in (False, True):
        for pre in (False, True):
            check(pkg, m, n, k, "bf16", bias=True, residual=residual, pre=pre, activation="relu")


def test_long_k_and_many_tiles(cuda, pkg):
    check(pkg, 16, 256, 16384, "bf16")
    check(pkg, 2100, 4104, 512, "bf16", bias=True, activation="silu", residual=True)
    check(pkg, 4096, 2048, 2048, "e4m3", out="bf16", scales=True)


@pytest.mark.parametrize("pair", [0, 256])
def test_infinities_and_nan_stay_in_their_rows_and_columns(cuda, pkg, tuning, pair):
    tuning("LINEAR_PAIR", pair)
    m, n, k = 40, 72, 136
    a, b, _, _ = operands(m, n, k, "bf16")
    a[3, 5], a[7, 9], b[11, 13] = float("nan"), float("inf"), float("inf")
    for activation in ("none", "relu"):
        c = torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")
        pkg.linear(m, n, k, pkg.BF16, a.data_ptr(), b.data_ptr(), pkg.BF16, c.data_ptr(), activation=d.act_code(pkg, activation))
        pkg.device_status()
        want = d.act(a.double() @ b.double(), activation)
        assert torch.equal(torch.isnan(c), torch.isnan(want)) and torch.equal(torch.isinf(c), torch.isinf(want))


def test_repeats_are_bit_identical(cuda, pkg, tuning):
    for pair, (m, n, k) in [(0, (16, 1032, 4096)), (0, (300, 264, 1024)), (256, (700, 1032, 512))]:
        tuning("LINEAR_PAIR", pair)
        first = check(pkg, m, n, k, "bf16", bias=True, residual=True)
        for _ in range(3):
            assert torch.equal(first, check(pkg, m, n, k, "bf16", bias=True, residual=True))


def layer_calls(pkg, s, stream):
    """A layer's training step: product with epilogue, its gradient, the two products of the backward pass."""
    m, n, k = s["m"], s["n"], s["k"]
    ptr = lambda key: s[key].data_ptr()  # noqa: E731
    pkg.linear(m, n, k, pkg.BF16, ptr("a"), ptr("b"), pkg.BF16, ptr("c"), bias=ptr("bias"), residual=ptr("residual"), pre=ptr("pre"),
               activation=pkg.ACT_GELU_TANH, stream=stream)
    pkg.epilogue_backward(m, n, pkg.BF16, ptr("dc"), ptr("pre"), pkg.ACT_GELU_TANH, ptr("dz"), ptr("dbias"), ptr("ws"), stream)
    pkg.linear(m, k, n, pkg.BF16, ptr("dz"), ptr("b"), pkg.BF16, ptr("da"), trans_b=1, stream=stream)
    pkg.linear(k, n, m, pkg.BF16, ptr("a"), ptr("dz"), pkg.BF16, ptr("db"), trans_a=1, stream=stream)


def layer_state(pkg, m, n, k, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda").bfloat16()  # noqa: E731
    empty = lambda *shape: torch.empty(shape, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    return {"m": m, "n": n, "k": k, "a": normal(m, k), "b": (normal(k, n).float() / k ** 0.5).bfloat16(), "bias": normal(n), "residual": normal(m, n),
            "dc": normal(m, n), "c": empty(m, n), "pre": empty(m, n), "dz": empty(m, n), "dbias": empty(n), "da": empty(m, k), "db": empty(k, n),
            "ws": torch.empty(pkg.epilogue_backward_workspace_bytes(m, n), dtype=torch.uint8, device="cuda")}


def layer_check(s):
    m, n, k = s["m"], s["n"], s["k"]
    u, a, b = d.half_step("bf16"), s["a"].double(), s["b"].double()
    dz = s["dc"].double() * d.act_grad(s["pre"].double(), "gelu_tanh")
    slope = 2.0 ** -20 * s["dc"].double().abs() * (1 + s["pre"].double().abs())
    d.assert_close(s["dz"], dz, u * dz.abs() + slope, "dZ")
    d.assert_close(s["dbias"], dz.sum(0), u * dz.sum(0).abs() + slope.sum(0) + m * 2.0 ** -24 * dz.abs().sum(0), "dbias")
    got = s["dz"].double()
    for key, want, mag, length in (("da", got @ b.t(), got.abs() @ b.abs().t(), n), ("db", a.t() @ got, a.abs().t() @ got.abs(), m)):
        off = d.sum_error(mag, length)
        d.assert_close(s[key], want, off + u * (want.abs() + off), key)


@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (9, 72, 136), (130, 264, 200), (520, 776, 1032)])
def test_layer_gradients(cuda, pkg, m, n, k):
    s = layer_state(pkg, m, n, k)
    if m % 8:      # dB = A^T dZ reads A as it lies, its rows being K long: any number of tokens
        assert k % 8 == 0
    layer_calls(pkg, s, 0)
    pkg.device_status()
    layer_check(s)


def test_layer_captured_and_replayed_on_another_stream(cuda, pkg):
    s = layer_state(pkg, 264, 520, 392)
    layer_calls(pkg, s, 0)
    torch.cuda.synchronize()
    keys = ("c", "pre", "dz", "dbias", "da", "db")
    want = {key: s[key].clone() for key in keys}
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        layer_calls(pkg, s, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        for key in keys:
            s[key].fill_(float("nan"))
        graph.replay()
    torch.cuda.synchronize()
    pkg.device_status()
    for key in keys:
        assert torch.equal(want[key], s[key]), key


def test_two_streams_at_once(cuda, pkg):
    states = [layer_state(pkg, 300, 520, 264, seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, st in zip(states, streams):
            layer_calls(pkg, s, st.cuda_stream)
    torch.cuda.synchronize()
    pkg.device_status()
    for s in states:
        layer_check(s)


def test_gradients_against_differences(cuda, pkg):
    """The slope of <dc, C> along a direction of A, by differences in 64 bits at the values that the layer used."""
    s = layer_state(pkg, 24, 40, 32)
    layer_calls(pkg, s, 0)
    torch.cuda.synchronize()
    a, b, dc = s["a"].double(), s["b"].double(), s["dc"].double()
    gen = torch.Generator(device="cuda").manual_seed(9)
    f = lambda x, w: (dc * d.act(x @ w + s["bias"].double(), "gelu_tanh")).sum()  # noqa: E731
    for key, at in (("da", a), ("db", b)):
        v = torch.randn(at.shape, generator=gen, device="cuda").double()
        h = 1e-5
        slope = (f(a + h * v, b) - f(a - h * v, b) if key == "da" else f(a, b + h * v) - f(a, b - h * v)) / (2 * h)
        got = (s[key].double() * v).sum()
        # bf16 roundings of pre, dZ and the gradient itself, each of half a step (of pre: times a second derivative of at most 1.2
        # and |pre| up to about 5), against the sum of magnitudes
        dz = s["dz"].double().abs()
        mag = (dz @ b.abs().t() * v.abs()).sum() if key == "da" else (a.abs().t() @ dz * v.abs()).sum()
        spread = (dc.abs() * s["pre"].double().abs() * 1.2) @ b.abs().t() if key == "da" else a.abs().t() @ (dc.abs() * s["pre"].double().abs() * 1.2)
        assert abs(got - slope) <= 2.0 ** -8 * (2 * mag + (spread * v.abs()).sum()), (key, got, slope)


def planted(t, trans, m, n, half, seed):
    """Operands in whose sums, at row 5 of every 32 and column 37 of every 64, the first half cancels the second and a small product of known sign is left over:
    (A and B as stored, both in 64 bits, rows, columns)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    k = 2 * half + 16
    a = torch.randn((m, k), generator=gen, device="cuda")
    b = torch.randn((k, n), generator=gen, device="cuda") * (1.0 if t == "e4m3" else k ** -0.5)
    if t == "e4m3":
        a, b = a * 16, b * 16
    a, b = a.to(d.TYPES[t]).float(), b.to(d.TYPES[t]).float()
    rows, cols = torch.arange(5, m, 32, device="cuda"), torch.arange(37, n, 64, device="cuda")
    a[rows, half:2 * half] = -a[rows, :half]
    b[half:2 * half, cols] = b[:half, cols]
    a[rows, 2 * half:] = 0.0
    b[2 * half:, cols] = 0.0
    # 2^-22 of values of size one: above fp16's smallest steps, below the tensor cores' error of such a sum (e4m3: 2^-10 of a sum of about 2^13)
    sign = torch.where(torch.rand((rows.numel(),), generator=gen, device="cuda") < 0.5, -1.0, 1.0)
    a[rows, 2 * half] = sign * (2.0 ** -5 if t == "e4m3" else 2.0 ** -11)
    b[2 * half, cols] = 2.0 ** -5 if t == "e4m3" else 2.0 ** -11
    a, b = a.to(d.TYPES[t]), b.to(d.TYPES[t])
    return (a.t().contiguous() if trans == "tn" else a, b.t().contiguous() if trans == "nt" else b, a.double(), b.double(), rows, cols)


@pytest.mark.parametrize("t,trans,half", [("f16", "nn", 512), ("f16", "nt", 2048), ("f16", "tn", 392), ("bf16", "nn", 2048), ("bf16", "tn", 512), ("bf16", "nt", 5000),
                                          ("e4m3", "nt", 2056)])
@pytest.mark.parametrize("m,n,bias", [(520, 264, False), (296, 1032, True), (8, 136, False)])
def test_relu_keeps_the_sign_of_sums_next_to_zero(cuda, pkg, t, trans, half, m, n, bias):
    """relu's slope is that of the sums as they are, not as the accumulation's cuts leave them: pre at the planted places is the 64-bit sum, rounded once, and
    dZ follows it."""
    out = "bf16" if t == "e4m3" else t
    ot = d.TYPES[out]
    a, b, a64, b64, rows, cols = planted(t, trans, m, n, half, half)
    k = a64.shape[1]
    bias_t = torch.randn(n, device="cuda").to(ot) if bias else None
    if bias:
        bias_t[cols] = 0
    sa = torch.rand(m, device="cuda") + 0.5 if t == "e4m3" else None
    c, p, dz = (torch.empty((m, n), dtype=ot, device="cuda") for _ in range(3))
    dc = torch.randn((m, n), device="cuda").to(ot)
    pkg.linear(m, n, k, d.code(pkg, t), a.data_ptr(), b.data_ptr(), d.code(pkg, out), c.data_ptr(), trans_a=int(trans == "tn"), trans_b=int(trans == "nt"),
               a_scale=0 if sa is None else sa.data_ptr(), bias=bias_t.data_ptr() if bias else 0, pre=p.data_ptr(), activation=pkg.ACT_RELU)
    pkg.epilogue_backward(m, n, d.code(pkg, out), dc.data_ptr(), p.data_ptr(), pkg.ACT_RELU, dz.data_ptr())
    pkg.device_status()
    z, want, mag = d.linear(a64, b64, sa, None, bias_t, "relu", None)
    off, u = d.sum_error(mag, k), d.half_step(out)
    d.assert_close(p, z, off + u * (z.abs() + off) + d.smallest(out), "pre")
    d.assert_close(c, want, off + u * (want.abs() + off) + d.smallest(out), "C")
    at = (rows[:, None], cols[None, :])
    assert bool((z[at] != 0).all())
    d.assert_close(p[at], z[at], u * 1.01 * z[at].abs() + d.smallest(out), "planted")
    assert torch.equal(dz[at], torch.where(z[at] > 0, dc[at], torch.zeros_like(dc[at])))


@pytest.mark.parametrize("t,trans,half", [("f16", "nn", 512), ("bf16", "nt", 2048), ("e4m3", "nt", 520)])
@pytest.mark.parametrize("m,n", [(6, 136), (294, 104), (38, 1064)])
def test_relu_border_in_few_rows(cuda, pkg, t, trans, half, m, n):
    """A piece of six rows, by itself and below others, where a column's size does not show; columns that end inside a piece."""
    test_relu_keeps_the_sign_of_sums_next_to_zero(cuda, pkg, t, trans, half, m // 8 * 8 if trans == "tn" else m, n, False)


def test_relu_border_captured_and_on_two_streams(cuda, pkg):
    """A captured product with new operands at every replay, beside one on another stream."""
    m, n, k = 296, 264, 1040
    sets = [planted("f16", "nn", m, n, 512, seed) for seed in range(4)]
    rows, cols = sets[0][4], sets[0][5]
    at = (rows[:, None], cols[None, :])
    a, b = sets[0][0].clone(), sets[0][1].clone()
    c, p, c2, p2 = (torch.empty((m, n), dtype=torch.float16, device="cuda") for _ in range(4))

    def call(x, w, to, pre, stream):
        pkg.linear(m, n, k, pkg.F16, x.data_ptr(), w.data_ptr(), pkg.F16, to.data_ptr(), pre=pre.data_ptr(), activation=pkg.ACT_RELU, stream=stream)
    want = []
    for s in sets:
        call(s[0], s[1], c, p, 0)
        pkg.device_status()
        assert torch.equal(p[at] > 0, (s[2] @ s[3])[at] > 0)
        want.append((c.clone(), p.clone()))
    side, other, graph = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(a, b, c, p, torch.cuda.current_stream().cuda_stream)
    for i, s in enumerate(sets):
        a.copy_(s[0]), b.copy_(s[1])
        torch.cuda.synchronize()
        graph.replay()
        call(sets[i - 1][0], sets[i - 1][1], c2, p2, other.cuda_stream)
        torch.cuda.synchronize()
        pkg.device_status()
        assert torch.equal(c, want[i][0]) and torch.equal(p, want[i][1]) and torch.equal(c2, want[i - 1][0]) and torch.equal(p2, want[i - 1][1])


def test_relu_border_beside_biases(cuda, pkg):
    """Sums that a bias of size one swallows are not the zeros of pruned blocks: elements next to zero in their rows and columns keep their side."""
    m, n = 296, 1032
    a, b, a64, b64, rows, cols = planted("f16", "nn", m, n, 512, 512)
    k, at = a64.shape[1], (rows[:, None], cols[None, :])
    sums = a64 @ b64
    for seed in range(20):
        bias = torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").half()
        bias[cols] = 0
        c, p = (torch.empty((m, n), dtype=torch.float16, device="cuda") for _ in range(2))
        pkg.linear(m, n, k, pkg.F16, a.data_ptr(), b.data_ptr(), pkg.F16, c.data_ptr(), bias=bias.data_ptr(), pre=p.data_ptr(), activation=pkg.ACT_RELU)
        pkg.device_status()
        assert torch.equal(p[at] > 0, sums[at] > 0), seed


def test_relu_border_of_many_tiles(cuda, pkg, tuning):
    """More elements next to the border than a warp keeps until its tiles are through."""
    tuning("LINEAR_PAIR", 64)
    m, n = 8000, 2048
    a, b, a64, b64, rows, cols = planted("f16", "nn", m, n, 264, 1)
    k = a64.shape[1]
    c, p = (torch.empty((m, n), dtype=torch.float16, device="cuda") for _ in range(2))
    pkg.linear(m, n, k, pkg.F16, a.data_ptr(), b.data_ptr(), pkg.F16, c.data_ptr(), pre=p.data_ptr(), activation=pkg.ACT_RELU)
    pkg.device_status()
    z, _, mag = d.linear(a64, b64)
    off, u, at = d.sum_error(mag, k), d.half_step("f16"), (rows[:, None], cols[None, :])
    d.assert_close(p, z, off + u * (z.abs() + off) + d.smallest("f16"), "pre")
    d.assert_close(p[at], z[at], u * 1.01 * z[at].abs() + d.smallest("f16"), "planted")


def test_relu_border_is_not_where_columns_are_small_or_empty(cuda, pkg):
    """Columns of tiny weights, of zeros, rows of zeros and of infinities beside ordinary ones: values as elsewhere, equal calls equal bits."""
    m, n, k = 300, 520, 776
    gen = torch.Generator(device="cuda").manual_seed(3)
    a = torch.randn((m, k), generator=gen, device="cuda").bfloat16()
    b = (torch.randn((k, n), generator=gen, device="cuda") / k ** 0.5).bfloat16()
    b[:, 3::8] *= 2.0 ** -30
    b[:, 5::8] = 0
    a[7], a[40:80] = 0, 0
    a[9, 11] = float("inf")
    got = []
    for _ in range(2):
        c, p = (torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        pkg.linear(m, n, k, pkg.BF16, a.data_ptr(), b.data_ptr(), pkg.BF16, c.data_ptr(), pre=p.data_ptr(), activation=pkg.ACT_RELU)
        pkg.device_status()
        got.append((c, p))
    rest = torch.arange(m, device="cuda") != 9
    z, want, mag = d.linear(a.double()[rest], b.double(), activation="relu")
    off, u = d.sum_error(mag, k), d.half_step("bf16")
    for c, p in got:
        d.assert_close(p[rest], z, off + u * (z.abs() + off), "pre")
        d.assert_close(c[rest], want, off + u * (want.abs() + off), "C")
        assert torch.equal(torch.isfinite(p[9]), torch.isfinite(a[9].double() @ b.double()))
    assert torch.equal(got[0][1].view(torch.int16), got[1][1].view(torch.int16))


def tail_error(z):
    """Relative error of the terms of gelu and its slope in 32 bits: the tail's fit 2.2e-7 (2 steps of 2^-23) and its evaluation 4 of them, the exponential 2 + 1.173 |x|
    at x = z^2 / 2 and its argument's roundings z^2; a few products: (z^2 1.6 + 11) 2^-23."""
    return (z * z + 8) * 2.0 ** -22


@pytest.mark.parametrize("pair", [0, 256])
@pytest.mark.parametrize("activation", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_activations_keep_their_negative_tail(cuda, pkg, tuning, t, activation, pair):
    """Values next to nothing, far left of zero, to the result's last bit: sums of one product are exact."""
    tuning("LINEAR_PAIR", pair)
    m, k = 72, 64
    # (smaller results than 2^-100 are no bf16 matter; gelu_tanh's fall faster)
    z = torch.linspace(-11.5 if activation == "gelu" else -8.5 if activation == "gelu_tanh" else -60, 6, m * k, device="cuda").view(m, k).to(d.TYPES[t])
    b, c = torch.eye(k, device="cuda").to(d.TYPES[t]), torch.empty((m, k), dtype=d.TYPES[t], device="cuda")
    pkg.linear(m, k, k, d.code(pkg, t), z.data_ptr(), b.data_ptr(), d.code(pkg, t), c.data_ptr(), activation=d.act_code(pkg, activation))
    pkg.device_status()
    want = d.act(z.double(), activation)
    # gelu_tanh's argument is a cube: a rounding of it counts about 2 u = 1.6 |z| (1 + 0.045 z^2) times, which is below 7 z^2 here
    e = tail_error(z.double()) * (1 if activation == "gelu" else 4)
    u = d.half_step(t)
    d.assert_close(c, want, (u + e * (1 + u)) * want.abs() + d.smallest(t), "C")


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_gelu_gradient_keeps_its_negative_tail(cuda, pkg, t):
    m, n = 72, 64
    z = torch.linspace(-11.5, 6, m * n, device="cuda").view(m, n).to(d.TYPES[t])
    dc, dz = torch.ones_like(z), torch.empty_like(z)
    pkg.epilogue_backward(m, n, d.code(pkg, t), dc.data_ptr(), z.data_ptr(), pkg.ACT_GELU, dz.data_ptr())
    pkg.device_status()
    z = z.double()
    want = d.act_grad(z, "gelu")
    terms = 0.5 * torch.special.erfc(-z / 2 ** 0.5) + z.abs() * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    off = tail_error(z) * terms
    d.assert_close(dz, want, off + d.half_step(t) * (want.abs() + off) + d.smallest(t), "dZ")


@pytest.mark.parametrize("m,n,k", [(24, 40, 32), (40, 24, 64)])
def test_gradients_against_differences_along_themselves(cuda, pkg, m, n, k):
    """The slope of <dc, C> along the signs of its gradient, by differences in 64 bits: a sum of the gradient's magnitudes, of which the roundings are a small share."""
    s = layer_state(pkg, m, n, k, seed=5)
    layer_calls(pkg, s, 0)
    pkg.device_status()
    a, b, dc, bias = s["a"].double(), s["b"].double(), s["dc"].double(), s["bias"].double()
    f = lambda x, w: (dc * d.act(x @ w + bias, "gelu_tanh")).sum()  # noqa: E731
    z = a @ b + bias
    slopes = dc * d.act_grad(z, "gelu_tanh")
    for key, grad in (("da", slopes @ b.t()), ("db", a.t() @ slopes)):
        v, h = torch.sign(grad), 1e-6
        slope = (f(a + h * v, b) - f(a - h * v, b) if key == "da" else f(a, b + h * v) - f(a, b - h * v)) / (2 * h)
        # half a step of bf16, 2^-8, each of pre (times a second derivative of at most 1.2), of dZ and of the gradient itself, against the sums of magnitudes
        share = 2.0 ** -8 * (slopes.abs() + dc.abs() * 1.2 * z.abs())
        tol = (share @ b.abs().t() if key == "da" else a.abs().t() @ share).sum() + 2.0 ** -8 * grad.abs().sum()
        assert tol <= 0.15 * slope.abs(), (key, tol, slope)
        assert abs((s[key].double() * v).sum() - slope) <= tol, (key, slope)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("activation", d.ACTS)
@pytest.mark.parametrize("m,n", [(1, 8), (9, 264), (1001, 520), (4100, 72)])
def test_epilogue_backward(cuda, pkg, t, activation, m, n):
    gen = torch.Generator(device="cuda").manual_seed(m)
    dc = torch.randn((m, n), generator=gen, device="cuda").to(d.TYPES[t])
    pre = (3 * torch.randn((m, n), generator=gen, device="cuda")).to(d.TYPES[t])
    dz, dz_ok = d.guarded(m, n, d.TYPES[t])
    db, db_ok = d.guarded(1, n, d.TYPES[t])
    ws = torch.empty(pkg.epilogue_backward_workspace_bytes(m, n), dtype=torch.uint8, device="cuda")
    pkg.epilogue_backward(m, n, d.code(pkg, t), dc.data_ptr(), pre.data_ptr() if activation != "none" else 0, d.act_code(pkg, activation),
                          dz.data_ptr(), db.data_ptr(), ws.data_ptr())
    pkg.device_status()
    want = dc.double() * d.act_grad(pre.double(), activation)
    # the slope: an exponential of up to 15 bits of argument, a quotient and a few 32-bit products
    off = 2.0 ** -20 * dc.double().abs() * (1 + pre.double().abs())
    u = d.half_step(t)
    d.assert_close(dz, want, u * want.abs() + off + d.smallest(t), "dZ")
    total = want.sum(0)
    d.assert_close(db[0], total, u * total.abs() + off.sum(0) + (m + 40) * 2.0 ** -24 * want.abs().sum(0) + d.smallest(t), "dbias")
    assert dz_ok() and db_ok()
    # in place, and each output alone
    alone = torch.empty_like(db[0])
    pkg.epilogue_backward(m, n, d.code(pkg, t), dc.data_ptr(), pre.data_ptr(), d.act_code(pkg, activation), 0, alone.data_ptr(), ws.data_ptr())
    pkg.epilogue_backward(m, n, d.code(pkg, t), dc.data_ptr(), pre.data_ptr(), d.act_code(pkg, activation), dc.data_ptr())
    pkg.device_status()
    assert torch.equal(alone, db[0]) and torch.equal(dc, dz)


def test_outputs_past_32_bit_offsets(cuda, pkg):
    """C, residual and gradients of more than 2^31 values: the last rows come out as they do by themselves."""
    m, n, k = 270000, 8192, 64
    a = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda")
    a[-200:] = torch.randn((200, k), device="cuda").bfloat16()
    b = torch.randn((k, n), device="cuda").bfloat16()
    c = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    c[-200:] = torch.randn((200, n), device="cuda").bfloat16()
    c[:-200] = 1.0
    res, small = c[-200:].clone(), torch.empty((200, n), dtype=torch.bfloat16, device="cuda")
    pkg.linear(m, n, k, pkg.BF16, a.data_ptr(), b.data_ptr(), pkg.BF16, c.data_ptr(), residual=c.data_ptr(), activation=pkg.ACT_SILU)
    pkg.linear(200, n, k, pkg.BF16, a[-200:].data_ptr(), b.data_ptr(), pkg.BF16, small.data_ptr(), residual=res.data_ptr(), activation=pkg.ACT_SILU)
    pkg.device_status()
    # (k = 64 is one run of additions in either kernel)
    assert torch.equal(c[-200:], small) and bool((c[:1000] == 1.0).all()) and bool((c[m // 2:m // 2 + 1000] == 1.0).all())
    ws = torch.empty(pkg.epilogue_backward_workspace_bytes(m, n), dtype=torch.uint8, device="cuda")
    db = torch.empty(n, dtype=torch.bfloat16, device="cuda")
    pkg.epilogue_backward(m, n, pkg.BF16, c.data_ptr(), c.data_ptr(), pkg.ACT_RELU, c.data_ptr(), db.data_ptr(), ws.data_ptr())
    pkg.epilogue_backward(200, n, pkg.BF16, small.data_ptr(), small.data_ptr(), pkg.ACT_RELU, small.data_ptr())
    pkg.device_status()
    assert torch.equal(c[-200:], small)
    total = small.double().sum(0) + (m - 200)
    d.assert_close(db, total, d.half_step("bf16") * total.abs() + 2.0 ** -20 * total.abs())
