"""CPU tests of the dense operators' entry points: constants of the binding, refusals before any device is touched, workspace sizes, and
the 64-bit restatements that the GPU tests compare with."""
import math
import os
import re

import pytest
import torch

import dense_ops as d

P = 4096          # an aligned address that is never read: validation fails first


def test_binding_agrees_with_the_header(pkg):
    hdr = open(pkg.HEADER_PATH).read()
    value = lambda name: int(re.search(rf"\b{name}\s*=\s*(\d+)", hdr).group(1))  # noqa: E731
    for name in ("F32", "F16", "BF16", "E4M3", "ACT_NONE", "ACT_RELU", "ACT_GELU", "ACT_GELU_TANH", "ACT_SILU"):
        assert getattr(pkg, name) == value("ESMM_" + name), name


def test_rmsnorm_refusals(pkg):
    L = pkg.lib()
    call = lambda M=4, K=64, t=pkg.BF16, x=P, res=0, w=P, s=0, ot=pkg.BF16, out=P, scale=0, rstd=0: L.esmm_rmsnorm(  # noqa: E731
        M, K, t, x, res, w, 1e-5, s, ot, out, scale, rstd, 0)
    assert call(x=0) == pkg.ERR_NULL and call(out=0) == pkg.ERR_NULL and call(ot=pkg.E4M3) == pkg.ERR_NULL
    assert call(M=0) == pkg.ERR_SHAPE and call(K=0) == pkg.ERR_SHAPE and call(M=-1) == pkg.ERR_SHAPE
    assert call(M=2 ** 31 - 1) == pkg.ERR_TOO_LARGE and call(K=2 ** 31 - 1) == pkg.ERR_TOO_LARGE
    assert call(t=pkg.E4M3) == pkg.ERR_UNSUPPORTED and call(t=17) == pkg.ERR_UNSUPPORTED
    assert call(ot=pkg.F16) == pkg.ERR_UNSUPPORTED and call(t=pkg.F32, ot=pkg.BF16) == pkg.ERR_UNSUPPORTED
    for bad in ({"x": P + 1}, {"res": P + 1}, {"w": P + 1}, {"s": P + 1}, {"out": P + 1}, {"rstd": P + 2}):
        assert call(**bad) == pkg.ERR_ALIGN, bad
    assert call(ot=pkg.E4M3, scale=P + 2) == pkg.ERR_ALIGN


def test_rmsnorm_backward_refusals(pkg):
    L = pkg.lib()
    call = lambda M=4, K=64, t=pkg.F16, g=P, h=P, w=P, r=P, s=0, dx=P, dw=P, ws=P: L.esmm_rmsnorm_backward(  # noqa: E731
        M, K, t, g, h, w, r, s, dx, dw, ws, 0)
    for bad in ({"g": 0}, {"h": 0}, {"r": 0}, {"dx": 0}, {"ws": 0}):
        assert call(**bad) == pkg.ERR_NULL, bad
    assert call(K=0) == pkg.ERR_SHAPE and call(M=0) == pkg.ERR_SHAPE
    assert call(K=2 ** 31 - 1) == pkg.ERR_TOO_LARGE
    assert call(t=pkg.E4M3) == pkg.ERR_UNSUPPORTED
    for bad in ({"g": P + 1}, {"h": P + 1}, {"w": P + 1}, {"s": P + 1}, {"dx": P + 1}, {"dw": P + 1}, {"r": P + 2}, {"ws": P + 8}):
        assert call(**bad) == pkg.ERR_ALIGN, bad


def test_quantize_refusals(pkg):
    L = pkg.lib()
    assert L.esmm_quantize_rows(4, 64, pkg.BF16, 0, P, P, 0) == pkg.ERR_NULL
    assert L.esmm_quantize_rows(4, 64, pkg.BF16, P, P, 0, 0) == pkg.ERR_NULL
    assert L.esmm_quantize_rows(0, 64, pkg.BF16, P, P, P, 0) == pkg.ERR_SHAPE
    assert L.esmm_quantize_rows(4, 64, pkg.E4M3, P, P, P, 0) == pkg.ERR_UNSUPPORTED
    assert L.esmm_quantize_rows(4, 64, pkg.F32, P + 2, P, P, 0) == pkg.ERR_ALIGN
    assert L.esmm_quantize_b(64, 8, pkg.F32, P, 0, P, 0) == pkg.ERR_NULL
    assert L.esmm_quantize_b(72, 8, pkg.F32, P, P, P, 0) == pkg.ERR_SHAPE       # K % 16
    assert L.esmm_quantize_b(64, 0, pkg.F32, P, P, P, 0) == pkg.ERR_SHAPE
    assert L.esmm_quantize_b(64, 8, pkg.E4M3, P, P, P, 0) == pkg.ERR_UNSUPPORTED
    assert L.esmm_quantize_b(64, 8, pkg.F32, P, P + 4, P, 0) == pkg.ERR_ALIGN
    assert L.esmm_quantize_b(65536 * 128, 8, pkg.F32, P, P, P, 0) == pkg.ERR_TOO_LARGE


def test_linear_refusals(pkg):
    L = pkg.lib()

    def call(M=16, N=64, K=64, t=pkg.BF16, a=P, ta=0, b=P, tb=0, ot=None, c=P, sa=0, sb=0, bias=0, res=0, pre=0, act=0):
        return L.esmm_linear(M, N, K, t, a, ta, b, tb, t if ot is None else ot, c, sa, sb, bias, res, pre, act, 0)
    for bad in ({"a": 0}, {"b": 0}, {"c": 0}):
        assert call(**bad) == pkg.ERR_NULL, bad
    for bad in ({"M": 0}, {"N": 0}, {"K": 0}, {"N": 60}, {"K": 60}, {"K": 60, "tb": 1}, {"M": 12, "ta": 1}, {"t": pkg.E4M3, "ot": pkg.BF16, "tb": 1, "K": 72}):
        assert call(**bad) == pkg.ERR_SHAPE, bad
    for bad in ({"t": pkg.F32}, {"t": 9}, {"ot": pkg.F16}, {"t": pkg.E4M3, "tb": 1}, {"t": pkg.E4M3, "ot": pkg.BF16}, {"ta": 1, "tb": 1},
                {"t": pkg.E4M3, "ot": pkg.BF16, "tb": 1, "ta": 1}, {"act": 5}, {"act": -1}):
        assert call(**bad) == pkg.ERR_UNSUPPORTED, bad
    for bad in ({"a": P + 8}, {"b": P + 8}, {"c": P + 8}, {"bias": P + 8}, {"res": P + 8}, {"pre": P + 8}, {"sa": P + 2}, {"sb": P + 2}):
        assert call(**bad) == pkg.ERR_ALIGN, bad
    assert call(M=2 ** 31 - 1) == pkg.ERR_TOO_LARGE


def test_epilogue_backward_refusals(pkg):
    L = pkg.lib()
    call = lambda M=4, N=64, t=pkg.BF16, g=P, z=P, act=pkg.ACT_SILU, dz=P, db=P, ws=P: L.esmm_epilogue_backward(  # noqa: E731
        M, N, t, g, z, act, dz, db, ws, 0)
    for bad in ({"g": 0}, {"z": 0}, {"dz": 0, "db": 0}, {"ws": 0}):
        assert call(**bad) == pkg.ERR_NULL, bad
    assert call(N=60) == pkg.ERR_SHAPE and call(N=6, t=pkg.F32) == pkg.ERR_SHAPE and call(M=0) == pkg.ERR_SHAPE
    assert call(t=pkg.E4M3) == pkg.ERR_UNSUPPORTED and call(act=7) == pkg.ERR_UNSUPPORTED
    for bad in ({"g": P + 8}, {"z": P + 8}, {"dz": P + 8}, {"db": P + 1}, {"ws": P + 8}):
        assert call(**bad) == pkg.ERR_ALIGN, bad
    assert call(M=2 ** 31 - 1) == pkg.ERR_TOO_LARGE


def test_helpers_raise_with_the_entry_points_name(pkg):
    with pytest.raises(pkg.EsmmError, match="esmm_linear") as e:
        pkg.linear(16, 60, 64, pkg.BF16, P, P, pkg.BF16, P)
    assert e.value.status == pkg.ERR_SHAPE
    with pytest.raises(pkg.EsmmError, match="esmm_rmsnorm"):
        pkg.rmsnorm(0, 64, pkg.BF16, P, 0, P, 1e-5, 0, pkg.BF16, P)


def test_workspace_sizes(pkg):
    assert pkg.rmsnorm_backward_workspace_bytes(1, 100) == 400
    for m in (7, 592, 100000):
        assert pkg.rmsnorm_backward_workspace_bytes(m, 64) == min(m, 592) * 64 * 4
    assert pkg.rmsnorm_backward_workspace_bytes(0, 64) == 0 and pkg.epilogue_backward_workspace_bytes(4, 0) == 0
    assert pkg.epilogue_backward_workspace_bytes(9, 64) == 2 * 64 * 4
    assert pkg.epilogue_backward_workspace_bytes(10 ** 6, 64) == 592 * 64 * 4


def test_tuning_hooks_are_known(pkg, tuning):
    for name in ("LINEAR_PAIR", "LINEAR_TAIL", "LINEAR_SPLIT", "LINEAR_COLUMNS"):
        tuning(name, 0)


@pytest.mark.parametrize("a", d.ACTS)
def test_slopes_are_those_of_the_activations(a):
    z = torch.linspace(-9, 9, 181, dtype=torch.float64) + 0.013      # (off the kink of relu)
    h = 1e-6
    slope = (d.act(z + h, a) - d.act(z - h, a)) / (2 * h)
    # third derivatives of up to about 2 times h^2, and 64-bit differences of values up to 9 over 2 h
    assert torch.allclose(slope, d.act_grad(z, a), rtol=0, atol=2 * h * h + 9 * 2.0 ** -52 / h)


def test_norm_restatement_against_autograd():
    gen = torch.Generator().manual_seed(1)
    x, res, w, dout, dsum = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((5, 12), (5, 12), (12,), (5, 12), (5, 12)))
    x.requires_grad_(), w.requires_grad_()
    h, rstd, y = d.norm(x, res, w, 1e-5)
    ((y * dout).sum() + (h * dsum).sum()).backward()
    dx, dw = d.norm_grad(dout, h.detach(), w.detach(), rstd.detach(), dsum)
    assert torch.allclose(x.grad, dx, rtol=1e-12, atol=1e-12) and torch.allclose(w.grad, dw, rtol=1e-12, atol=1e-12)
    assert math.isclose(d.row_scale(torch.zeros(1, 3, dtype=torch.float64))[0].item(), 2.0 ** -100 / 448)


def sources(pkg):
    root = os.path.join(os.path.dirname(pkg.__file__), "csrc")
    return {f: open(os.path.join(root, f)).read() for f in sorted(os.listdir(root)) if f.endswith((".cu", ".cuh"))}


def test_loads_of_what_other_threads_store_stay_behind_their_barriers(pkg):
    """A shared-memory load in inline assembly reads what others have stored: unless it is volatile, as the barriers are, the compiler may move it across them."""
    loads = [(name, m) for name, text in sources(pkg).items() for m in re.findall(r'asm[^"]*"ld\.shared[^"]*"', text)]
    assert len(loads) >= 2
    for name, m in loads:
        assert m.startswith("asm volatile"), (name, m)


def test_a_warp_agrees_on_its_wait_before_its_tensor_core_instructions(pkg):
    """A bounded wait may pass in one lane and run out in another; what is the whole warp's (sync.aligned) comes only after a vote."""
    text = sources(pkg)["esmm_linear.cu"]
    waits = [m.start() for m in re.finditer(r"[^_]mbar_wait\(", text)]
    assert len(waits) >= 6
    for at in waits:
        after = re.search(r"linear_tmem_ld\(|linear_mma_step<|linear_load_step<|linear_commit<", text[at:])
        assert after is None or "__all_sync" in text[text.rfind("\n", 0, at):at + after.start()], text[at:at + 60]


def test_every_row_kernel_is_checked_in_the_checked_build(pkg):
    """Kernels whose indices depend on the sizes have bounds checks for -DESMM_CHECKED, each kind of access under a number of its own."""
    text = sources(pkg)["esmm_rows.cu"]
    kernels = text.split("__global__")[1:]
    assert len(kernels) == 10
    for body in kernels:
        body = body[:body.index("\n}\n")]
        assert "bounds_ok(" in body, body.split("\n")[1]
