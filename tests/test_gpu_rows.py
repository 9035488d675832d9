"""GPU tests of the norm with the residual's addition, its gradients and the e4m3 forms of rows and weights, against 64 bits."""
import pytest
import torch

import dense_ops as d

pytestmark = pytest.mark.gpu
EPS = 1e-5


def tensors(m, k, t, seed=0, offset=0):
    """x, residual, weight, dout, dsum; `offset` elements off a 16-byte boundary"""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def one(rows, std=1.0, mean=0.0):
        flat = torch.empty((rows * k + offset,), dtype=d.TYPES[t], device="cuda")
        view = flat[offset:].view(rows, k)
        view.copy_(torch.randn((rows, k), generator=gen, device="cuda") * std + mean)
        return view
    return one(m), one(m, 2.0), one(1, 0.2, 1.0)[0], one(m, 0.1), one(m, 0.1)


def norm_tolerance(k):
    """relative error of rstd and of y before rounding: a 32-bit sum of k squares over up to 1024 threads, a square root, a few products"""
    return (k / 256 + 24) * 2.0 ** -24


ROWS = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 100), (9, 509), (1, 4096), (17, 4096), (1300, 256), (1300, 1024), (2000, 136), (3, 16384), (2, 40000), (4, 9001),
        (1, 20011), (1400, 1501), (1200, 100)]


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,k", ROWS)
def test_norm(cuda, pkg, t, m, k):
    x, res, w, _, _ = tensors(m, k, t)
    for residual, weight in ((res, w), (None, w), (res, None)):
        h, h_ok = d.guarded(m, k, d.TYPES[t])
        out, out_ok = d.guarded(m, k, d.TYPES[t])
        rstd, rstd_ok = d.guarded(1, m, torch.float32)
        pkg.rmsnorm(m, k, d.code(pkg, t), x.data_ptr(), 0 if residual is None else residual.data_ptr(), 0 if weight is None else weight.data_ptr(), EPS,
                    h.data_ptr(), d.code(pkg, t), out.data_ptr(), 0, rstd.data_ptr())
        pkg.device_status()
        h64, r64, y64 = d.norm(x, residual, weight, EPS)
        u, e = d.half_step(t), norm_tolerance(k)
        d.assert_close(h, h64, (u + 2.0 ** -24) * h64.abs() + d.smallest(t), "h")
        d.assert_close(rstd[0], r64, e * r64, "rstd")
        # (h itself is a 32-bit sum of two: off by half a step of it, also where it nearly cancels)
        inner = (e * y64.abs() + 2.0 ** -24 * y64.abs())
        d.assert_close(out, y64, inner + u * (y64.abs() + inner) + d.smallest(t), "out")
        assert h_ok() and out_ok() and rstd_ok()


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,k", ROWS)
def test_norm_to_e4m3(cuda, pkg, t, m, k):
    x, res, w, _, _ = tensors(m, k, t, seed=1)
    out, out_ok = d.guarded(m, k, torch.float8_e4m3fn)
    scale, scale_ok = d.guarded(1, m, torch.float32)
    pkg.rmsnorm(m, k, d.code(pkg, t), x.data_ptr(), res.data_ptr(), w.data_ptr(), EPS, 0, pkg.E4M3, out.data_ptr(), scale.data_ptr())
    pkg.device_status()
    _, _, y64 = d.norm(x, res, w, EPS)
    check_e4m3(out, scale[0], y64, norm_tolerance(k) + 2.0 ** -24)
    assert out_ok() and scale_ok()


def check_e4m3(out, scale, y64, e):
    want = d.row_scale(y64)
    d.assert_close(scale, want, (e + 4 * 2.0 ** -24) * want, "scale")
    # half a step of e4m3 (relative 2^-4, below 2^-6 the spacing is 2^-9), and what y and the scale are off
    q = y64 / want[:, None]
    off = (2 * e + 8 * 2.0 ** -24) * q.abs()
    d.assert_close(out.float(), q, off + torch.maximum((2.0 ** -4) * (q.abs() + off), torch.full_like(q, 2.0 ** -10)), "codes")


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,k", ROWS)
def test_quantize_rows(cuda, pkg, t, m, k):
    x, _, _, _, _ = tensors(m, k, t, seed=2)
    x[0].zero_()
    out, out_ok = d.guarded(m, k, torch.float8_e4m3fn)
    scale, scale_ok = d.guarded(1, m, torch.float32)
    pkg.quantize_rows(m, k, d.code(pkg, t), x.data_ptr(), out.data_ptr(), scale.data_ptr())
    pkg.device_status()
    check_e4m3(out, scale[0], x.double(), 0.0)
    assert not out[0].float().any() and scale[0, 0] > 0
    assert out_ok() and scale_ok()


def test_special_values(cuda, pkg):
    """A row of zeros, infinities and NaN, in each kind of result."""
    m, k = 6, 200
    x = torch.randn((m, k), device="cuda").bfloat16()
    x[0].zero_()
    x[2, 3], x[3, 5], x[4, 7] = float("nan"), float("inf"), -float("inf")
    out = torch.empty_like(x)
    rstd, scale = torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
    pkg.rmsnorm(m, k, pkg.BF16, x.data_ptr(), 0, 0, EPS, 0, pkg.BF16, out.data_ptr(), 0, rstd.data_ptr())
    pkg.device_status()
    assert not out[0].any() and abs(rstd[0].item() - EPS ** -0.5) < 1e-3 * EPS ** -0.5
    assert out[2].isnan().all() and rstd[2].isnan()
    for r, c in ((3, 5), (4, 7)):     # mean square infinite: rstd 0, infinity times 0 in its place and zeros elsewhere
        assert out[r, c].isnan() and rstd[r] == 0 and not out[r][torch.arange(k, device="cuda") != c].any()
    assert torch.isfinite(out[1]).all() and torch.isfinite(out[5]).all()
    q = torch.empty((m, k), dtype=torch.float8_e4m3fn, device="cuda")
    pkg.quantize_rows(m, k, pkg.BF16, x.data_ptr(), q.data_ptr(), scale.data_ptr())
    pkg.device_status()
    f = q.float()
    assert f[2, 3].isnan() and torch.isfinite(f[2]).sum() == k - 1      # the rest of the row keeps its own scale
    assert scale[3].isinf() and f[3, 5].isnan()
    huge = torch.full((1, 16), 3e38, device="cuda")
    huge[0, 3] = 1e-30
    pkg.quantize_rows(1, 16, pkg.F32, huge.data_ptr(), q.data_ptr(), scale.data_ptr())
    pkg.device_status()
    assert (q.view(-1)[:16].float() == 448.0).sum() == 15


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("m,k", [(3, 64), (2000, 512), (5, 1501), (2, 40000)])
def test_norm_in_place(cuda, pkg, t, m, k):
    x, res, w, _, _ = tensors(m, k, t, seed=4)
    h, out, rstd = torch.empty_like(x), torch.empty_like(x), torch.empty(m, device="cuda")
    c = d.code(pkg, t)
    pkg.rmsnorm(m, k, c, x.data_ptr(), res.data_ptr(), w.data_ptr(), EPS, h.data_ptr(), c, out.data_ptr(), 0, rstd.data_ptr())
    pkg.rmsnorm(m, k, c, x.data_ptr(), res.data_ptr(), w.data_ptr(), EPS, res.data_ptr(), c, x.data_ptr())
    pkg.device_status()
    assert torch.equal(res, h) and torch.equal(x, out)


@pytest.mark.parametrize("offset", [1, 3])
def test_norm_unaligned(cuda, pkg, offset):
    for t in ("bf16", "f32"):
        x, res, w, dout, dsum = tensors(12, 512, t, seed=5, offset=offset)
        a = [v.clone() for v in (x, res, w, dout, dsum)]
        got = []
        for (xx, rr, ww, gg, ss) in ((x, res, w, dout, dsum), a):
            h, out, rstd, dx, dw = (torch.empty((12, 512), dtype=d.TYPES[t], device="cuda"), torch.empty((12, 512), dtype=d.TYPES[t], device="cuda"),
                                    torch.empty(12, device="cuda"), torch.empty((12, 512), dtype=d.TYPES[t], device="cuda"),
                                    torch.empty(512, dtype=d.TYPES[t], device="cuda"))
            c = d.code(pkg, t)
            ws = torch.empty(pkg.rmsnorm_backward_workspace_bytes(12, 512), dtype=torch.uint8, device="cuda")
            pkg.rmsnorm(12, 512, c, xx.data_ptr(), rr.data_ptr(), ww.data_ptr(), EPS, h.data_ptr(), c, out.data_ptr(), 0, rstd.data_ptr())
            pkg.rmsnorm_backward(12, 512, c, gg.data_ptr(), h.data_ptr(), ww.data_ptr(), rstd.data_ptr(), ss.data_ptr(), dx.data_ptr(), dw.data_ptr(),
                                 ws.data_ptr())
            pkg.device_status()
            got.append((h, out, dx, dw))
        # (sums in another order: a step of the type at most)
        assert torch.equal(got[0][0], got[1][0])
        for p, q in zip(got[0][1:], got[1][1:]):
            d.assert_close(p, q.double(), 2 * d.half_step(t) * q.double().abs() * 1.01 + 1e-5 * q.double().abs().max())


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,k", ROWS)
def test_norm_backward(cuda, pkg, t, m, k):
    x, _, w, dout, dsum = tensors(m, k, t, seed=6)
    _, r64, _ = d.norm(x, None, w, EPS)
    rstd = r64.float()
    c, u = d.code(pkg, t), d.half_step(t)
    ws = torch.empty(pkg.rmsnorm_backward_workspace_bytes(m, k), dtype=torch.uint8, device="cuda")
    for weight, add in ((w, dsum), (None, None)):
        dx, dx_ok = d.guarded(m, k, d.TYPES[t])
        dw, dw_ok = d.guarded(1, k, d.TYPES[t])
        pkg.rmsnorm_backward(m, k, c, dout.data_ptr(), x.data_ptr(), 0 if weight is None else weight.data_ptr(), rstd.data_ptr(),
                             0 if add is None else add.data_ptr(), dx.data_ptr(), dw.data_ptr(), ws.data_ptr())
        pkg.device_status()
        want, want_w = d.norm_grad(dout, x, weight, rstd, add)
        # 32-bit products and the row's sum of products, against the magnitudes that enter
        xh = (x.double() * rstd.double()[:, None]).abs()
        gw = dout.double().abs() * (1.0 if weight is None else weight.double().abs())
        mag = rstd.double()[:, None] * (gw + xh * (gw * xh).mean(dim=1, keepdim=True)) + (0 if add is None else add.double().abs())
        off = (k / 256 + 24) * 2.0 ** -24 * mag
        d.assert_close(dx, want, off + u * (want.abs() + off) + d.smallest(t), "dx")
        mag_w = (dout.double().abs() * xh).sum(dim=0)
        off = (m + 40) * 2.0 ** -24 * mag_w
        d.assert_close(dw[0], want_w, off + u * (want_w.abs() + off) + d.smallest(t), "dweight")
        assert dx_ok() and dw_ok()
        again = torch.empty_like(dw[0])
        pkg.rmsnorm_backward(m, k, c, dout.data_ptr(), x.data_ptr(), 0 if weight is None else weight.data_ptr(), rstd.data_ptr(),
                             0 if add is None else add.data_ptr(), dx.data_ptr(), again.data_ptr(), ws.data_ptr())
        pkg.device_status()
        assert torch.equal(again, dw[0])
    # over its own input, and without the weight's gradient
    dx2 = torch.empty_like(x)
    pkg.rmsnorm_backward(m, k, c, dout.data_ptr(), x.data_ptr(), w.data_ptr(), rstd.data_ptr(), dsum.data_ptr(), dx2.data_ptr())
    pkg.rmsnorm_backward(m, k, c, dout.data_ptr(), x.data_ptr(), w.data_ptr(), rstd.data_ptr(), dsum.data_ptr(), dsum.data_ptr())
    pkg.device_status()
    assert torch.equal(dx2, dsum)


# Many more rows than are under way in a CTA at once: one warp per row, a CTA per row that keeps it in registers, one that reads its slot again (16-bit K past 8192, FP32
# past 4096), and rows that are no whole vectors with four, eight and sixteen elements per thread.
MANY_ROWS = [(40000, 64), (20000, 512), (5000, 4096), (1500, 8192), (1500, 16384), (5000, 1501), (2500, 4001), (1300, 6091)]


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,k", MANY_ROWS)
def test_norm_backward_of_many_rows(cuda, pkg, t, m, k):
    test_norm_backward(cuda, pkg, t, m, k)


@pytest.mark.parametrize("m,k", MANY_ROWS)
def test_norm_backward_of_many_rows_over_its_inputs(cuda, pkg, m, k):
    test_norm_backward_over_its_inputs(cuda, pkg, m, k)


def test_norm_gradient_against_differences(cuda, pkg):
    m, k = 6, 96
    x, _, w, dout, _ = tensors(m, k, "f32", seed=7)
    _, r64, _ = d.norm(x, None, w, EPS)
    rstd, dx, dw = r64.float(), torch.empty_like(x), torch.empty(k, device="cuda")
    ws = torch.empty(pkg.rmsnorm_backward_workspace_bytes(m, k), dtype=torch.uint8, device="cuda")
    pkg.rmsnorm_backward(m, k, pkg.F32, dout.data_ptr(), x.data_ptr(), w.data_ptr(), rstd.data_ptr(), 0, dx.data_ptr(), dw.data_ptr(), ws.data_ptr())
    pkg.device_status()
    f = lambda xx, ww: (dout.double() * d.norm(xx, None, ww, EPS)[2]).sum()  # noqa: E731
    h = 1e-5
    for at, got in ((x, dx), (w, dw)):
        v = torch.randn_like(at).double()
        up, down = (f(x.double() + h * v, w), f(x.double() - h * v, w)) if at is x else (f(x, w.double() + h * v), f(x, w.double() - h * v))
        slope = (up - down) / (2 * h)
        # differences of second order in h = 1e-5 (about 1e-10 of the values), 32-bit gradients
        assert abs((got.double() * v).sum() - slope) <= 1e-5 * (got.double() * v).abs().sum() + 1e-8


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("k,n", [(16, 1), (16, 33), (272, 100), (1040, 264), (4096, 7)])
def test_quantize_b(cuda, pkg, t, k, n):
    b = torch.randn((k, n), device="cuda").to(d.TYPES[t])
    b[:, 0].zero_()
    bt, bt_ok = d.guarded(n, k, torch.float8_e4m3fn)
    scale, scale_ok = d.guarded(1, n, torch.float32)
    pkg.quantize_b(k, n, d.code(pkg, t), b.data_ptr(), bt.data_ptr(), scale.data_ptr())
    pkg.device_status()
    check_e4m3(bt, scale[0], b.double().t(), 0.0)
    assert not bt[0].float().any()
    assert bt_ok() and scale_ok()


@pytest.mark.parametrize("m", [1, 16, 200])
def test_feed_forward_block_in_8_bits(cuda, pkg, m):
    """Norm, up-projection with its activation, rows in 8 bits again, down-projection plus the residual stream, as they are used."""
    k, n = 528, 1040
    gen = torch.Generator(device="cuda").manual_seed(m)
    normal = lambda *shape, std=1.0: (torch.randn(shape, generator=gen, device="cuda") * std).bfloat16()  # noqa: E731
    x, res, w = normal(m, k), normal(m, k), (1 + normal(k, std=0.2))
    b1, b2, bias = normal(k, n, std=k ** -0.5), normal(n, k, std=n ** -0.5), normal(n, std=0.1)
    e4m3, f32 = dict(dtype=torch.float8_e4m3fn, device="cuda"), dict(dtype=torch.float32, device="cuda")
    bt1, s1, bt2, s2 = torch.empty((n, k), **e4m3), torch.empty(n, **f32), torch.empty((k, n), **e4m3), torch.empty(k, **f32)
    pkg.quantize_b(k, n, pkg.BF16, b1.data_ptr(), bt1.data_ptr(), s1.data_ptr())
    pkg.quantize_b(n, k, pkg.BF16, b2.data_ptr(), bt2.data_ptr(), s2.data_ptr())
    q1, r1, q2, r2 = torch.empty((m, k), **e4m3), torch.empty(m, **f32), torch.empty((m, n), **e4m3), torch.empty(m, **f32)
    u, out = torch.empty((m, n), dtype=torch.bfloat16, device="cuda"), torch.empty((m, k), dtype=torch.bfloat16, device="cuda")
    h = res.clone()
    pkg.rmsnorm(m, k, pkg.BF16, x.data_ptr(), h.data_ptr(), w.data_ptr(), EPS, h.data_ptr(), pkg.E4M3, q1.data_ptr(), r1.data_ptr())
    pkg.linear(m, n, k, pkg.E4M3, q1.data_ptr(), bt1.data_ptr(), pkg.BF16, u.data_ptr(), trans_b=1, a_scale=r1.data_ptr(), b_scale=s1.data_ptr(),
               bias=bias.data_ptr(), activation=pkg.ACT_GELU)
    pkg.quantize_rows(m, n, pkg.BF16, u.data_ptr(), q2.data_ptr(), r2.data_ptr())
    pkg.linear(m, k, n, pkg.E4M3, q2.data_ptr(), bt2.data_ptr(), pkg.BF16, out.data_ptr(), trans_b=1, a_scale=r2.data_ptr(), b_scale=s2.data_ptr(),
               residual=h.data_ptr())
    pkg.device_status()
    # each step against the values that the step before left
    h64, _, y64 = d.norm(x, res, w, EPS)
    d.assert_close(h, h64, (d.half_step("bf16") + 2.0 ** -24) * h64.abs())
    check_e4m3(q1, r1, y64, norm_tolerance(k) + 2.0 ** -24)
    ub = d.half_step("bf16")
    z, want, mag = d.linear(q1.double(), bt1.double().t(), r1, s1, bias, "gelu", None)
    off = 1.13 * d.sum_error(mag, k) + 2.0 ** -20 * z.abs()
    d.assert_close(u, want, off + ub * (want.abs() + off))
    check_e4m3(q2, r2, u.double(), 0.0)
    _, want, mag = d.linear(q2.double(), bt2.double().t(), r2, s2, None, "none", h)
    off = d.sum_error(mag, n) + 2.0 ** -20 * want.abs()
    d.assert_close(out, want, off + ub * (want.abs() + off))


def test_pointers_that_a_call_does_not_use_may_lie_anywhere(cuda, pkg):
    """d_scale without e4m3, d_workspace without the weight's or bias's gradient, d_pre without an activation."""
    m, k = 12, 64
    x, _, w, dout, _ = tensors(m, k, "bf16", seed=9)
    odd = torch.zeros(4096, dtype=torch.uint8, device="cuda")[1:].data_ptr()
    rstd = torch.empty(m, device="cuda")
    got = []
    for unused in (0, odd):
        out, dx, dz = (torch.empty_like(x) for _ in range(3))
        pkg.rmsnorm(m, k, pkg.BF16, x.data_ptr(), 0, w.data_ptr(), EPS, 0, pkg.BF16, out.data_ptr(), unused, rstd.data_ptr())
        pkg.rmsnorm_backward(m, k, pkg.BF16, dout.data_ptr(), x.data_ptr(), w.data_ptr(), rstd.data_ptr(), 0, dx.data_ptr(), 0, unused)
        pkg.epilogue_backward(m, k, pkg.BF16, dout.data_ptr(), unused, pkg.ACT_NONE, dz.data_ptr(), 0, unused)
        pkg.device_status()
        got.append((out, dx, dz))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_norm_captured_and_replayed_with_new_inputs(cuda, pkg):
    m, k = 300, 1032
    sets = [tensors(m, k, "bf16", seed=s) for s in (11, 12)]
    x, res, w, dout, dsum = (v.clone() for v in sets[0])
    h, out, dx = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    q, scale, rstd = torch.empty((m, k), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
    dw = torch.empty_like(w)
    ws = torch.empty(pkg.rmsnorm_backward_workspace_bytes(m, k), dtype=torch.uint8, device="cuda")

    def calls(stream):
        pkg.rmsnorm(m, k, pkg.BF16, x.data_ptr(), res.data_ptr(), w.data_ptr(), EPS, h.data_ptr(), pkg.BF16, out.data_ptr(), 0, rstd.data_ptr(), stream)
        pkg.rmsnorm_backward(m, k, pkg.BF16, dout.data_ptr(), h.data_ptr(), w.data_ptr(), rstd.data_ptr(), dsum.data_ptr(), dx.data_ptr(), dw.data_ptr(),
                             ws.data_ptr(), stream)
        pkg.quantize_rows(m, k, pkg.BF16, out.data_ptr(), q.data_ptr(), scale.data_ptr(), stream)
    outputs = (h, out, rstd, dx, dw, q.view(torch.uint8), scale)
    want = []
    for s in sets:
        for to, v in zip((x, res, w, dout, dsum), s):
            to.copy_(v)
        calls(0)
        torch.cuda.synchronize()
        want.append([o.clone() for o in outputs])
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        calls(torch.cuda.current_stream().cuda_stream)
    for s, expected in zip(sets, want):
        for to, v in zip((x, res, w, dout, dsum), s):
            to.copy_(v)
        for o in outputs:
            o.zero_()
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        for o, e in zip(outputs, expected):
            assert torch.equal(o, e)
    pkg.device_status()


def test_norms_on_two_streams_at_once(cuda, pkg):
    m, k = 700, 2048
    runs = []
    for seed in (21, 22):
        x, res, w, dout, dsum = tensors(m, k, "bf16", seed=seed)
        runs.append(dict(x=x, res=res, w=w, dout=dout, dsum=dsum, h=torch.empty_like(x), out=torch.empty_like(x), dx=torch.empty_like(x), dw=torch.empty_like(w),
                         rstd=torch.empty(m, device="cuda"), ws=torch.empty(pkg.rmsnorm_backward_workspace_bytes(m, k), dtype=torch.uint8, device="cuda"),
                         stream=torch.cuda.Stream()))

    def go(r, stream):
        p = {key: v.data_ptr() for key, v in r.items() if key != "stream"}
        pkg.rmsnorm(m, k, pkg.BF16, p["x"], p["res"], p["w"], EPS, p["h"], pkg.BF16, p["out"], 0, p["rstd"], stream)
        pkg.rmsnorm_backward(m, k, pkg.BF16, p["dout"], p["h"], p["w"], p["rstd"], p["dsum"], p["dx"], p["dw"], p["ws"], stream)
    want = []
    for r in runs:
        go(r, 0)
        torch.cuda.synchronize()
        want.append([r[key].clone() for key in ("h", "out", "dx", "dw")])
    for _ in range(20):
        for r in runs:
            go(r, r["stream"].cuda_stream)
    torch.cuda.synchronize()
    pkg.device_status()
    for r, e in zip(runs, want):
        for key, v in zip(("h", "out", "dx", "dw"), e):
            assert torch.equal(r[key], v)


@pytest.mark.parametrize("m,k", [(40, 512), (40, 1501), (3, 12000), (2, 40000)])
def test_norm_backward_over_its_inputs(cuda, pkg, m, k):
    x, _, w, dout, dsum = tensors(m, k, "bf16", seed=8)
    rstd = d.norm(x, None, w, EPS)[1].float()
    want = torch.empty_like(x)
    call = lambda g, s, to: pkg.rmsnorm_backward(m, k, pkg.BF16, g.data_ptr(), x.data_ptr(), w.data_ptr(), rstd.data_ptr(), s.data_ptr(), to.data_ptr())  # noqa: E731
    call(dout, dsum, want)
    over = dout.clone()
    call(over, dsum, over)
    call(dout, dsum, dsum)
    pkg.device_status()
    assert torch.equal(over, want) and torch.equal(dsum, want)


def test_rows_past_32_bit_offsets(cuda, pkg):
    """More than 2^31 elements: the last rows come out as they do by themselves."""
    m, k = 70000, 32768
    x = torch.empty((m, k), dtype=torch.bfloat16, device="cuda")
    x.fill_(0.5)
    x[-3:] = torch.randn((3, k), device="cuda").bfloat16()
    out, rstd, scale = torch.empty_like(x), torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
    pkg.rmsnorm(m, k, pkg.BF16, x.data_ptr(), 0, 0, EPS, 0, pkg.BF16, out.data_ptr(), 0, rstd.data_ptr())
    small, r = torch.empty((3, k), dtype=torch.bfloat16, device="cuda"), torch.empty(3, device="cuda")
    # (one or four vectors per thread: sums in another order, a step of the type at most)
    pkg.rmsnorm(3, k, pkg.BF16, x[-3:].data_ptr(), 0, 0, EPS, 0, pkg.BF16, small.data_ptr(), 0, r.data_ptr())
    pkg.device_status()
    assert torch.allclose(rstd[-3:], r, rtol=1e-6) and bool((out[:5].float() == 1.0).all())
    d.assert_close(out[-3:], small.double(), 2 * d.half_step("bf16") * small.double().abs() * 1.01)
    dx, dsmall = out, torch.empty_like(small)                  # the gradient over its own input's buffer
    dx[-3:] = small
    pkg.rmsnorm_backward(m, k, pkg.BF16, dx.data_ptr(), x.data_ptr(), 0, rstd.data_ptr(), 0, dx.data_ptr())
    pkg.rmsnorm_backward(3, k, pkg.BF16, small.data_ptr(), x[-3:].data_ptr(), 0, rstd[-3:].data_ptr(), 0, dsmall.data_ptr())
    q, qs = torch.empty((m, k), dtype=torch.uint8, device="cuda"), torch.empty((3, k), dtype=torch.uint8, device="cuda")
    pkg.quantize_rows(m, k, pkg.BF16, x.data_ptr(), q.data_ptr(), scale.data_ptr())
    pkg.quantize_rows(3, k, pkg.BF16, x[-3:].data_ptr(), qs.data_ptr(), r.data_ptr())
    pkg.device_status()
    assert torch.equal(dx[-3:], dsmall) and torch.equal(q[-3:], qs) and torch.equal(scale[-3:], r)
