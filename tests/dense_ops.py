"""The dense operators restated in 64 bits (norm, products with epilogue, e4m3 rows and their gradients), and their tolerances.

Every tolerance counts roundings: half a step of the result's type (eps / 2 relative to the value), 32-bit sums, nothing else."""
import math

import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
E4M3_MAX, TINY = 448.0, 2.0 ** -100


def code(pkg, t):
    return {"f32": pkg.F32, "f16": pkg.F16, "bf16": pkg.BF16, "e4m3": pkg.E4M3}[t]


def act_code(pkg, a):
    return {"none": pkg.ACT_NONE, "relu": pkg.ACT_RELU, "gelu": pkg.ACT_GELU, "gelu_tanh": pkg.ACT_GELU_TANH, "silu": pkg.ACT_SILU}[a]


def half_step(t):
    return torch.finfo(TYPES[t]).eps / 2


def smallest(t):
    """half the spacing of the type's smallest numbers"""
    return torch.finfo(TYPES[t]).smallest_normal * torch.finfo(TYPES[t]).eps / 2


def act(z, a):
    if a == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if a == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2.0))
    if a == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if a == "silu":
        return z * torch.sigmoid(z)
    return z


def act_grad(z, a):
    if a == "relu":
        return (z > 0).to(z.dtype)
    if a == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if a == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        s = torch.sigmoid(2 * c * (z + 0.044715 * z ** 3))
        return s + z * s * (1 - s) * 2 * c * (1 + 3 * 0.044715 * z * z)
    if a == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def norm(x, residual, weight, eps):
    """(h, rstd, y)"""
    h = x.double() if residual is None else x.double() + residual.double()
    rstd = 1 / torch.sqrt((h * h).mean(dim=1) + eps)
    y = h * rstd[:, None]
    return h, rstd, y if weight is None else y * weight.double()


def norm_grad(dout, h, weight, rstd, dsum):
    """(dx, dweight)"""
    xh, g = h.double() * rstd.double()[:, None], dout.double()
    gw = g if weight is None else g * weight.double()
    dx = rstd.double()[:, None] * (gw - xh * (gw * xh).mean(dim=1, keepdim=True))
    return dx if dsum is None else dx + dsum.double(), (g * xh).sum(dim=0)


def row_scale(y):
    return y.abs().amax(dim=1).clamp(min=TINY) / E4M3_MAX


def linear(a, b, a_scale=None, b_scale=None, bias=None, activation="none", residual=None):
    """(z, C, sum of |products|): a is M x K, b K x N in 64 bits"""
    z, mag = a @ b, a.abs() @ b.abs()
    if a_scale is not None:
        z, mag = z * a_scale.double()[:, None], mag * a_scale.double()[:, None]
    if b_scale is not None:
        z, mag = z * b_scale.double()[None, :], mag * b_scale.double()[None, :]
    if bias is not None:
        z, mag = z + bias.double(), mag + bias.double().abs()
    c = act(z, activation)
    return z, c if residual is None else c + residual.double(), mag


def sum_error(mag, k):
    """What FP32 accumulation may be off: the tensor core adds 16 (32 in 8 bits) products at a time to its sum, aligned to the largest
    of them: two steps of 2^-23 of the magnitudes per addition, and a few for the parts of K and the epilogue's own additions."""
    return (k / 16 + 16) * 2.0 ** -22 * mag


def guarded(rows, cols, dtype, device="cuda", margin=512):
    """A rows x cols view (16-byte aligned) inside a buffer of a known pattern, and a function that tells whether the margins are intact."""
    size = torch.empty((), dtype=dtype).element_size()
    n = rows * cols * size
    n16 = -(-n // 16) * 16
    raw = torch.full((margin + n16 + margin,), 0xA5, dtype=torch.uint8, device=device)
    view = raw[margin:margin + n].view(dtype).view(rows, cols)

    def intact():
        return bool((raw[:margin] == 0xA5).all()) and bool((raw[margin + n:] == 0xA5).all())
    return view, intact


def assert_close(got, want, tol, what=""):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), got[bad][:4].tolist(), want[bad][:4].tolist(), (got - want).abs()[bad].max().item())
