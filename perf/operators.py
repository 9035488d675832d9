"""The dense operators around a pruned layer as timed cases: root-mean-square norm with the residual's addition (forward with a
16-bit, FP32 or 8-bit result, and backward), the matrix product with scales, bias, activation and residual in its epilogue (forward
for one token up to a long prompt, and the training step with its gradients), and a whole 8-bit feed-forward block.

Every case names
  op       "norm"       h = x + residual; out = h / rms(h) * weight, in the inputs' type or in e4m3 with one scale per row
           "norm_train" the same in the inputs' type, and its gradients
           "linear"     C = act(a_scale b_scale (A B) + bias) + residual
           "linear_train"  C with the values before the activation kept, then dZ and dbias, dA = dZ B^T, dB = A^T dZ
           "block8"     norm to e4m3, up-projection with activation, e4m3 per row again, down-projection plus residual
  dtype    "bf16", "fp16", "fp32" (norms), "e4m3" (products: A per row, B per column scaled, B stored transposed; bf16 results)
  m, k, n  tokens, width of A, width of C
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
E4M3_MAX = 448.0
TINY = 2.0 ** -100          # smallest amax that a row's scale is made from
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}


def _norm(name, dtype, out, m, k, residual=True):
    return {"name": name, "op": "norm", "dtype": dtype, "out": out, "m": m, "k": k, "residual": residual}


def _norm_train(name, dtype, m, k, residual=True):
    return {"name": name, "op": "norm_train", "dtype": dtype, "m": m, "k": k, "residual": residual}


def _linear(name, dtype, m, k, n, act, bias, residual):
    return {"name": name, "op": "linear", "dtype": dtype, "m": m, "k": k, "n": n, "act": act, "bias": bias, "residual": residual}


def _linear_train(name, dtype, m, k, n, act, bias=True, residual=True):
    return {"name": name, "op": "linear_train", "dtype": dtype, "m": m, "k": k, "n": n, "act": act, "bias": bias,
            "residual": residual}


def listed():
    return [
        # one new token before a layer: launch latency and nothing else
        _norm("norm_token", "bf16", "bf16", 1, 4096),
        # the same step on a prompt, feeding an 8-bit product
        _norm("norm_prompt_e4m3", "bf16", "e4m3", 2048, 4096),
        # training: a batch of tokens, forward and backward
        _norm_train("norm_train", "bf16", 8192, 4096),
        # odd sizes in FP32: rows that no vector load divides
        _norm_train("norm_train_odd", "fp32", 1003, 1509),
        # decoding: 16 token rows through the up-projection
        _linear("up_16", "bf16", 16, 4096, 11008, "silu", True, False),
        # one token through the 8-bit down-projection: the weights' bytes and nothing else
        _linear("down_1_e4m3", "e4m3", 1, 11008, 4096, "none", False, True),
        # a prompt through the up-projection
        _linear("up_prompt", "bf16", 2048, 4096, 11008, "gelu", True, False),
        # a prompt through the 8-bit down-projection
        _linear("down_prompt_e4m3", "e4m3", 2048, 11008, 4096, "none", True, True),
        # no size a multiple of a tile
        _linear("ragged_fp16", "fp16", 1000, 2008, 1512, "gelu_tanh", True, True),
        # training steps of a projection: a large one, and one of a small model
        _linear_train("train_large", "bf16", 2048, 4096, 11008, "silu"),
        _linear_train("train_small", "fp16", 520, 776, 1032, "relu"),
        # a whole 8-bit feed-forward block of a short prompt
        {"name": "block_e4m3", "op": "block8", "dtype": "e4m3", "m": 512, "k": 4096, "n": 11008, "act": "gelu_tanh"},
    ]


def _log_int(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v // step * step))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_train", "linear", "linear", "linear", "linear_train", "block8"])
    if op in ("norm", "norm_train"):
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        case = {"op": op, "dtype": dtype, "m": _log_int(rng, 1, 8192), "k": _log_int(rng, 64, 16384, rng.choice([1, 8, 64])),
                "residual": rng.random() < 0.75}
        while case["m"] * case["k"] > 8192 * 4096:
            case["m"] = max(1, case["m"] // 2)
        if op == "norm":
            case["out"] = rng.choice([dtype, "e4m3"])
        return case
    dtype = "e4m3" if op == "block8" else rng.choice(["bf16", "fp16"] if op == "linear_train" else ["bf16", "fp16", "e4m3", "e4m3"])
    while True:
        case = {"op": op, "dtype": dtype, "m": _log_int(rng, 1, 4096), "k": _log_int(rng, 128, 11008, 16),
                "n": _log_int(rng, 128, 11008, 16 if op == "block8" else 8), "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])}
        if op != "block8":
            case["bias"], case["residual"] = rng.random() < 0.5, rng.random() < 0.5
        if case["m"] * case["k"] * case["n"] <= 2048 * 4096 * 11008:
            return case


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _e4m3_rows(x):
    """x of FP32 as e4m3 with one scale per row."""
    scale = x.abs().amax(dim=1, keepdim=True).clamp(min=TINY) / E4M3_MAX
    return (x / scale).to(torch.float8_e4m3fn), scale[:, 0].contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, m, k, n = case["op"], case["m"], case["k"], case.get("n", 0)
    t = TYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).add_(mean)

    def empty(*shape, dtype):
        return torch.empty(shape, dtype=dtype, device="cuda")

    s = {"case": case}
    if op in ("norm", "norm_train"):
        # activations with a few wide channels, as a residual stream has them
        wide = 1.0 + 8.0 * (torch.rand((k,), generator=gen, device="cuda") < 0.01).float()
        s["x"] = normal(m, k).mul_(wide).to(t)
        s["residual"] = normal(m, k, std=2.0).to(t) if case["residual"] else None
        s["weight"] = normal(k, std=0.2, mean=1.0).to(t)
        s["rstd"] = empty(m, dtype=torch.float32)
        s["h"] = empty(m, k, dtype=t) if case["residual"] else None
        if op == "norm":
            s["out"] = empty(m, k, dtype=TYPES[case["out"]])
            s["scale"] = empty(m, dtype=torch.float32)
        else:
            s["out"], s["dx"] = empty(m, k, dtype=t), empty(m, k, dtype=t)
            s["dout"] = normal(m, k, std=0.1).to(t)
            s["dh"] = normal(m, k, std=0.1).to(t) if case["residual"] else None
            s["dweight"] = empty(k, dtype=t)
            s["workspace"] = empty(1024 * k, dtype=torch.float32)
        return s
    if op == "block8":
        # weights of both projections in e4m3, transposed, one scale per output column
        s["x"], s["residual"] = normal(m, k).to(torch.bfloat16), normal(m, k, std=2.0).to(torch.bfloat16)
        s["weight"] = normal(k, std=0.2, mean=1.0).to(torch.bfloat16)
        s["b1"], s["b1_scale"] = _e4m3_rows(normal(n, k, std=1.0 / math.sqrt(k)))
        s["b2"], s["b2_scale"] = _e4m3_rows(normal(k, n, std=1.0 / math.sqrt(n)))
        s["bias1"] = normal(n, std=0.1).to(torch.bfloat16)
        s["h"], s["out"] = empty(m, k, dtype=torch.bfloat16), empty(m, k, dtype=torch.bfloat16)
        s["q1"], s["s1"] = empty(m, k, dtype=torch.float8_e4m3fn), empty(m, dtype=torch.float32)
        s["u"] = empty(m, n, dtype=torch.bfloat16)
        s["q2"], s["s2"] = empty(m, n, dtype=torch.float8_e4m3fn), empty(m, dtype=torch.float32)
        return s
    out = torch.bfloat16 if case["dtype"] == "e4m3" else t
    if case["dtype"] == "e4m3":
        s["a"], s["a_scale"] = _e4m3_rows(normal(m, k))
        s["b"], s["b_scale"] = _e4m3_rows(normal(n, k, std=1.0 / math.sqrt(k)))
    else:
        s["a"] = normal(m, k).to(t)
        s["b"] = normal(k, n, std=1.0 / math.sqrt(k)).to(t)
    s["bias"] = normal(n, std=0.1).to(out) if case["bias"] else None
    s["residual"] = normal(m, n).to(out) if case["residual"] else None
    s["c"] = empty(m, n, dtype=out)
    if op == "linear_train":
        s["pre"], s["dz"] = empty(m, n, dtype=out), empty(m, n, dtype=out)
        s["dc"] = normal(m, n, std=0.1).to(out)
        s["dbias"] = empty(n, dtype=out) if case["bias"] else None
        s["da"], s["db"] = empty(m, k, dtype=out), empty(k, n, dtype=out)
        s["workspace"] = empty(1024 * n, dtype=torch.float32)
    return s


# ---- the plain forms: 32 bits, rounded once at the end of each operator ------------------------------------------------
_SQRT_HALF, _GELU_C, _GELU_A = math.sqrt(0.5), math.sqrt(2.0 / math.pi), 0.044715


def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0.0)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * _SQRT_HALF))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(_GELU_C * (z + _GELU_A * z * z * z)))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return sig * (1.0 + z * (1.0 - sig))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * _SQRT_HALF)) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        th = torch.tanh(_GELU_C * (z + _GELU_A * z * z * z))
        return 0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * _GELU_C * (1.0 + 3.0 * _GELU_A * z * z)
    return torch.ones_like(z)


def _plain_norm(x, residual, weight):
    """(h, rstd, out) in FP32"""
    h = x.float()
    if residual is not None:
        h = h + residual.float()
    rstd = 1.0 / torch.sqrt((h * h).sum(dim=1) / h.shape[1] + EPS)
    return h, rstd, h * rstd[:, None] * weight.float()


def _plain_linear(a, b, a_scale, b_scale, bias, act, residual):
    """(values before the activation, C) in FP32; b is K x N"""
    z = a @ b
    if a_scale is not None:
        z = z * a_scale[:, None] * b_scale[None, :]
    if bias is not None:
        z = z + bias.float()
    c = _act(z, act)
    if residual is not None:
        c = c + residual.float()
    return z, c


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op in ("norm", "norm_train"):
        t = s["x"].dtype
        h, rstd, out = _plain_norm(s["x"], s["residual"], s["weight"])
        stored = h.to(t)
        if op == "norm":
            got = {"rstd": rstd}
            if case["out"] == "e4m3":
                got["out"], got["scale"] = _e4m3_rows(out)
            else:
                got["out"] = out.to(t)
            if case["residual"]:
                got["h"] = stored
            return got
        # the backward pass reads the stored h
        xhat, g = stored.float() * rstd[:, None], s["dout"].float()
        gw = g * s["weight"].float()
        dx = rstd[:, None] * (gw - xhat * ((gw * xhat).sum(dim=1) / h.shape[1])[:, None])
        if s["dh"] is not None:
            dx = dx + s["dh"].float()
        got = {"out": out.to(t), "rstd": rstd, "dx": dx.to(t), "dweight": (g * xhat).sum(dim=0).to(t)}
        if case["residual"]:
            got["h"] = stored
        return got
    if op == "block8":
        h, _, out = _plain_norm(s["x"], s["residual"], s["weight"])
        q1, s1 = _e4m3_rows(out)
        _, u = _plain_linear(q1.float(), s["b1"].float().t(), s1, s["b1_scale"], s["bias1"], case["act"], None)
        u = u.to(torch.bfloat16)
        q2, s2 = _e4m3_rows(u.float())
        h = h.to(torch.bfloat16)
        _, c = _plain_linear(q2.float(), s["b2"].float().t(), s2, s["b2_scale"], None, "none", h)
        return {"h": h, "u": u, "out": c.to(torch.bfloat16)}
    a, b = s["a"].float(), s["b"].float()
    scaled = case["dtype"] == "e4m3"
    z, c = _plain_linear(a, b.t() if scaled else b, s.get("a_scale"), s.get("b_scale"), s["bias"], case["act"], s["residual"])
    c = c.to(s["c"].dtype)
    if op == "linear":
        return c
    t = s["c"].dtype
    pre = z.to(t)
    dz = s["dc"].float() * _act_grad(pre.float(), case["act"])
    got = {"c": c, "pre": pre, "dz": dz.to(t)}
    if case["bias"]:
        got["dbias"] = dz.sum(dim=0).to(t)
    dz = dz.to(t).float()
    got["da"], got["db"] = (dz @ b.t()).to(t), (a.t() @ dz).to(t)
    return got


# ---- the framework's calls -----------------------------------------------------------------------------------------------
def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _own(s):
    from __graft_entry__ import load_package
    pkg = load_package()
    case = s["case"]
    op, m, k, n = case["op"], case["m"], case["k"], case.get("n", 0)
    types = {"bf16": pkg.BF16, "fp16": pkg.F16, "fp32": pkg.F32, "e4m3": pkg.E4M3}
    t = types[case["dtype"]]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "norm":
        e4m3 = case["out"] == "e4m3"
        pkg.rmsnorm(m, k, t, _ptr(s["x"]), _ptr(s["residual"]), _ptr(s["weight"]), EPS, _ptr(s["h"]), types[case["out"]],
                    _ptr(s["out"]), _ptr(s["scale"]) if e4m3 else 0, _ptr(s["rstd"]), stream)
        got = {"rstd": s["rstd"], "out": s["out"]}
        if e4m3:
            got["scale"] = s["scale"]
        if case["residual"]:
            got["h"] = s["h"]
        return got
    if op == "norm_train":
        h = s["x"] if s["h"] is None else s["h"]
        pkg.rmsnorm(m, k, t, _ptr(s["x"]), _ptr(s["residual"]), _ptr(s["weight"]), EPS, _ptr(s["h"]), t, _ptr(s["out"]), 0,
                    _ptr(s["rstd"]), stream)
        pkg.rmsnorm_backward(m, k, t, _ptr(s["dout"]), _ptr(h), _ptr(s["weight"]), _ptr(s["rstd"]), _ptr(s["dh"]), _ptr(s["dx"]),
                             _ptr(s["dweight"]), _ptr(s["workspace"]), stream)
        got = {"out": s["out"], "rstd": s["rstd"], "dx": s["dx"], "dweight": s["dweight"]}
        if case["residual"]:
            got["h"] = s["h"]
        return got
    act = {"none": pkg.ACT_NONE, "relu": pkg.ACT_RELU, "gelu": pkg.ACT_GELU, "gelu_tanh": pkg.ACT_GELU_TANH, "silu": pkg.ACT_SILU}[case["act"]]
    if op == "block8":
        pkg.rmsnorm(m, k, pkg.BF16, _ptr(s["x"]), _ptr(s["residual"]), _ptr(s["weight"]), EPS, _ptr(s["h"]), pkg.E4M3, _ptr(s["q1"]),
                    _ptr(s["s1"]), 0, stream)
        pkg.linear(m, n, k, pkg.E4M3, _ptr(s["q1"]), _ptr(s["b1"]), pkg.BF16, _ptr(s["u"]), trans_b=1, a_scale=_ptr(s["s1"]),
                   b_scale=_ptr(s["b1_scale"]), bias=_ptr(s["bias1"]), activation=act, stream=stream)
        pkg.quantize_rows(m, n, pkg.BF16, _ptr(s["u"]), _ptr(s["q2"]), _ptr(s["s2"]), stream)
        pkg.linear(m, k, n, pkg.E4M3, _ptr(s["q2"]), _ptr(s["b2"]), pkg.BF16, _ptr(s["out"]), trans_b=1, a_scale=_ptr(s["s2"]),
                   b_scale=_ptr(s["b2_scale"]), residual=_ptr(s["h"]), stream=stream)
        return {"h": s["h"], "u": s["u"], "out": s["out"]}
    scaled = case["dtype"] == "e4m3"
    out = pkg.BF16 if scaled else t
    pkg.linear(m, n, k, t, _ptr(s["a"]), _ptr(s["b"]), out, _ptr(s["c"]), trans_b=1 if scaled else 0, a_scale=_ptr(s.get("a_scale")),
               b_scale=_ptr(s.get("b_scale")), bias=_ptr(s["bias"]), residual=_ptr(s["residual"]), pre=_ptr(s.get("pre")),
               activation=act, stream=stream)
    if op == "linear":
        return s["c"]
    pkg.epilogue_backward(m, n, t, _ptr(s["dc"]), _ptr(s["pre"]), act, _ptr(s["dz"]), _ptr(s["dbias"]), _ptr(s["workspace"]), stream)
    pkg.linear(m, k, n, t, _ptr(s["dz"]), _ptr(s["b"]), t, _ptr(s["da"]), trans_b=1, stream=stream)
    pkg.linear(k, n, m, t, _ptr(s["a"]), _ptr(s["dz"]), t, _ptr(s["db"]), trans_a=1, stream=stream)
    got = {"c": s["c"], "pre": s["pre"], "dz": s["dz"], "da": s["da"], "db": s["db"]}
    if case["bias"]:
        got["dbias"] = s["dbias"]
    return got


def run(s):
    return _own(s) if own else _plain(s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}


def work(case):
    op, m, k, n = case["op"], case["m"], case["k"], case.get("n", 0)
    size = _BYTES[case["dtype"]]
    if op == "norm":
        res = 2 if case["residual"] else 0                       # residual in, sum out
        scales = 4.0 * m if case["out"] == "e4m3" else 0.0
        return {"bytes": m * k * (size * (1 + res) + _BYTES[case["out"]]) + k * size + 4.0 * m + scales, "flops": 5.0 * m * k}
    if op == "norm_train":
        res = 3 if case["residual"] else 0                       # residual in, sum out, the sum's gradient in
        # x, out; dout, dx, h again
        return {"bytes": m * k * size * (5.0 + res) + 3.0 * k * size + 8.0 * m, "flops": 15.0 * m * k}
    if op == "block8":
        # x, residual, h out and in, out; u is written and read and its e4m3 form too
        return {"bytes": 2.0 * k * n + m * k * (2.0 * 5 + 2.0) + m * n * (2.0 * 2 + 2.0), "flops": 4.0 * m * k * n}
    out = 2.0
    once = size * (m * k + k * n) + out * m * n * (2 if case["residual"] else 1)
    if op == "linear":
        return {"bytes": once + (out * n if case["bias"] else 0), "flops": 2.0 * m * k * n}
    # pre out and in, dC in, dZ out and in twice; B and A again; dA, dB out
    return {"bytes": once + out * m * n * 6 + size * 2.0 * (m * k + k * n), "flops": 6.0 * m * k * n}


# ---- the same from the definition in 64 bits ------------------------------------------------------------------------------
def _act64(z, act):
    """(value, derivative) in 64 bits"""
    if act == "relu":
        on = z > 0
        return torch.where(on, z, torch.zeros_like(z)), on.double()
    if act == "silu":
        sig = torch.special.expit(z)
        return z * sig, sig + z * sig * (1.0 - sig)
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        return z * cdf, cdf + z * torch.exp(-z * z / 2.0) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        # (1 + tanh u) / 2 is the logistic function of 2 u
        c = math.sqrt(2.0 / math.pi)
        sig = torch.special.expit(2.0 * c * (z + 0.044715 * z ** 3))
        return z * sig, sig + z * sig * (1.0 - sig) * 2.0 * c * (1.0 + 3.0 * 0.044715 * z ** 2)
    return z, torch.ones_like(z)


def _rows64(y):
    scale = torch.clamp(torch.linalg.vector_norm(y, ord=math.inf, dim=1), min=2.0 ** -100) / 448.0
    return (y / scale[:, None]).float().to(torch.float8_e4m3fn), scale


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]

    def wide(key):
        return None if s.get(key) is None else s[key].double()

    if op in ("norm", "norm_train", "block8"):
        x, r, w = wide("x"), wide("residual"), wide("weight")
        h = x if r is None else x + r
        rstd = torch.rsqrt(torch.linalg.vector_norm(h, dim=1) ** 2 / case["k"] + EPS)
        y = torch.einsum("mk,m,k->mk", h, rstd, w)
        kept = h.to(s["x"].dtype).double()
    if op == "norm":
        got = {"rstd": rstd, "out": y}
        if case["out"] == "e4m3":
            got["out"], got["scale"] = _rows64(y)
            got["out"] = got["out"].double()
        if case["residual"]:
            got["h"] = h
        return got
    if op == "norm_train":
        xh, g = torch.einsum("mk,m->mk", kept, rstd), wide("dout")
        inner = torch.einsum("mk,k,mk->m", g, w, xh) / case["k"]
        dx = torch.einsum("mk,k,m->mk", g, w, rstd) - torch.einsum("mk,m,m->mk", xh, inner, rstd)
        if s["dh"] is not None:
            dx = dx + wide("dh")
        got = {"out": y, "rstd": rstd, "dx": dx, "dweight": torch.einsum("mk,mk->k", g, xh)}
        if case["residual"]:
            got["h"] = h
        return got
    if op == "block8":
        q, sc = _rows64(y)
        z = torch.einsum("mk,nk,m,n->mn", q.double(), wide("b1"), sc, wide("b1_scale")) + wide("bias1")
        u = _act64(z, case["act"])[0]
        q, sc = _rows64(u.to(torch.bfloat16).double())
        c = torch.einsum("mk,nk,m,n->mn", q.double(), wide("b2"), sc, wide("b2_scale"))
        return {"h": h, "u": u, "out": c + kept}
    a, b = wide("a"), wide("b")
    if case["dtype"] == "e4m3":
        z = torch.einsum("mk,nk->mn", a, b)
        z = torch.einsum("mn,m,n->mn", z, wide("a_scale"), wide("b_scale"))
    else:
        z = torch.einsum("mk,kn->mn", a, b)
    if s["bias"] is not None:
        z = z + wide("bias")
    c = _act64(z, case["act"])[0]
    if s["residual"] is not None:
        c = c + wide("residual")
    if op == "linear":
        return c
    t = s["c"].dtype
    dz = wide("dc") * _act64(z.to(t).double(), case["act"])[1]
    got = {"c": c, "pre": z, "dz": dz}
    if case["bias"]:
        got["dbias"] = dz.sum(dim=0)
    dz = dz.to(t).double()
    got["da"], got["db"] = torch.einsum("mn,kn->mk", dz, b), torch.einsum("mk,mn->kn", a, dz)
    return got
