"""Cases of the microscaled operators: MXFP8 and MXFP4 quantisation, the RMSNorm
with the residual's addition and the gated GELU that end in it, and the products
with an MXFP4 weight.

A case is a dict of plain values; `op` names the call:

  quantize  mx_quantize of [m][k] values, f32 or bf16, read back with mx_dequantize
  norm      add_rmsnorm_mx of m rows: h = residual + x (x normed first where `post`), MX(rmsnorm(h)), and h
  gelu      gelu_mul_mx of m rows of a fused gate|up output
  linear    qlinear_forward (mxfp4_gemv where m = 1 and there is no bias) of m rows of f32 activations
  rows      mxfp4_gemm of m rows of bf16 activations
  mx        mx_gemm of m rows of MXFP8 or MXFP4 activations, f32 or bf16 out

Microscaled tensors are planar: the elements of [rows][k] (e4m3 bytes, or e2m1
codes two to a byte, the even element low), then one e8m0 byte for each 32 of a
row.  Their values are exact in bf16, in which the 8- and 4-bit outputs are given.

Hidden and feed-forward widths are those of Gemma-3 4B (2560, 10240) and 1B
(1152, 6912).  Weights have a standard deviation of 1/sqrt(k); hidden states have
a few channels that are many times the others, as trained models' do.
"""
from __future__ import annotations

import importlib.util
import math
import pathlib
import sys

import torch

own = False

REPO = pathlib.Path(__file__).resolve().parents[1]
PKG_DIR = REPO / "rich-triplet_amd"
DEV = "cuda:0"
EPS = 1e-6
EMAX = {"mx8": 8, "mx4": 2}      # exponent of the largest power of two an element holds
LARGEST = {"mx8": 448.0, "mx4": 6.0}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _package():
    if "rich_triplet_amd" not in sys.modules:
        spec = importlib.util.spec_from_file_location("rich_triplet_amd", PKG_DIR / "__init__.py",
                                                      submodule_search_locations=[str(PKG_DIR)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["rich_triplet_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["rich_triplet_amd"]


def listed():
    return [
        # one token's hidden state on its way into an 8-bit product
        dict(name="quantize_token", op="quantize", m=1, k=2560, src="f32", fmt="mx8"),
        # a bf16 feed-forward weight made an MXFP4 one at load
        dict(name="quantize_weight", op="quantize", m=10240, k=2560, src="bf16", fmt="mx4"),
        # between two sublayers of a decode step
        dict(name="norm_token", op="norm", m=1, k=2560, post=True, fmt="mx8"),
        # the same of a prompt chunk
        dict(name="norm_prompt", op="norm", m=4096, k=2560, post=True, fmt="mx8"),
        # the feed-forward activation of a verify batch, 4-bit
        dict(name="gelu_verify", op="gelu", m=5, k=6912, src="f32", fmt="mx4"),
        # of a prompt chunk, from a bf16 gate|up product
        dict(name="gelu_prompt", op="gelu", m=4096, k=10240, src="bf16", fmt="mx8"),
        # a decode step's gate projection
        dict(name="linear_token", op="linear", m=1, n=10240, k=2560, bias=False),
        # a verify batch on an output of odd width, with a bias
        dict(name="linear_verify", op="linear", m=5, n=2561, k=6912, bias=True),
        # a prompt's down projection with activations kept in f32
        dict(name="linear_prompt", op="linear", m=512, n=2560, k=10240, bias=False),
        # a short ragged prompt in bf16
        dict(name="rows_prompt", op="rows", m=77, n=10240, k=2560),
        # a short prompt's down projection on 8-bit activations
        dict(name="mx_short", op="mx", m=300, n=2560, k=10240, fmt="mx8", out="f32", bias=False),
        # gate|up of two prompt chunks on 4-bit activations
        dict(name="mx_prompt", op="mx", m=8192, n=20480, k=2560, fmt="mx4", out="bf16", bias=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "norm", "gelu", "linear", "rows", "mx"])
    k = 32 * _log(rng, 2, 320)
    fmt = rng.choice(["mx8", "mx4"])
    if op in ("quantize", "norm", "gelu"):
        m = _log(rng, 1, 8192)
        more = dict(post=rng.random() < 0.5) if op == "norm" else dict(src=rng.choice(["f32", "bf16"]))
        return dict(op=op, m=m, k=k, fmt=fmt, **more)
    n = _log(rng, 100, 20480)
    if op == "mx":
        return dict(op=op, m=_log(rng, 1, 8192 if k <= 2560 else 2048), n=n, k=k, fmt=fmt,
                    out=rng.choice(["f32", "bf16"]), bias=rng.random() < 0.5)
    m = _log(rng, 1, 1024)
    return dict(op="linear", m=m, n=n, k=k, bias=rng.random() < 0.5) if op == "linear" else dict(op=op, m=m, n=n, k=k)


def work(case):
    m, k, op = case["m"], case["k"], case["op"]
    size = {"f32": 4, "bf16": 2, "mx8": 1 + 1 / 32, "mx4": 0.5 + 1 / 32}
    if op == "quantize":
        return dict(bytes=m * k * (size[case["src"]] + 2), flops=2 * m * k)
    if op == "norm":
        return dict(bytes=m * k * (4 + 4 + 4 + 2) + 8 * k, flops=(12 if case["post"] else 7) * m * k)
    if op == "gelu":
        return dict(bytes=m * k * (2 * size[case["src"]] + 2), flops=12 * m * k)
    n = case["n"]
    a = size["f32" if op == "linear" else "bf16" if op == "rows" else case["fmt"]]
    c = size[case.get("out", "f32")]
    return dict(bytes=n * k * size["mx4"] + m * k * a + m * n * c + (4 * n if case.get("bias") else 0),
                flops=2 * m * n * k)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _power(e, bits, bias, whole, real):
    """2^e for integers e of a type's normal range, exactly: the exponent field alone."""
    return ((e.to(whole) + bias) << bits).view(real)


def _planar(x, fmt):
    """The planar microscaled tensor of x [rows][k], by comparisons and the type's own rounding."""
    rows, k = x.shape
    b = x.float().reshape(rows, k // 32, 32)
    top = b.abs().amax(-1)
    byte = (top.view(torch.int32) >> 23).sub(EMAX[fmt]).clamp(0, 254)
    v = (b * _power(127 - byte, 23, 127, torch.int32, torch.float32).unsqueeze(-1)).reshape(rows, k)
    if fmt == "mx8":
        codes = v.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).reshape(-1)
    else:
        c = _e2m1_code(v)
        codes = (c[:, 0::2] | (c[:, 1::2] << 4)).reshape(-1)
    return torch.cat([codes, byte.to(torch.uint8).reshape(-1)])


def _e2m1_code(v):
    """Nearest e2m1 code of v, ties to the even code, by comparisons with the middles."""
    a = v.abs()
    c = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    return c | ((v < 0).to(torch.uint8) << 3)


def _values(planar, fmt, rows, k):
    """f32 values of a planar microscaled tensor."""
    n = rows * k if fmt == "mx8" else rows * k // 2
    if fmt == "mx8":
        e = planar[:n].view(torch.float8_e4m3fn).float()
    else:
        half = torch.tensor(E2M1, device=planar.device)
        table = torch.cat([half, -half])
        e = torch.stack([table[(planar[:n] & 15).int()], table[(planar[:n] >> 4).int()]], -1)
    byte = planar[n:].int().reshape(-1, 1)
    scale = torch.where(byte > 0, byte << 23, 1 << 22).view(torch.float32)  # 2^(byte - 127), at byte 0 a subnormal
    return (e.reshape(-1, 32) * scale).reshape(rows, k)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    m, k, op = case["m"], case["k"], case["op"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    def hidden(rows, width):
        channel = torch.where(torch.rand(width, generator=gen, device=DEV) < 0.01, 20.0, 1.0)
        return normal(rows, width) * channel * torch.exp(0.3 * normal(rows, 1))

    s = dict(case=case)
    if op == "quantize":
        s["x"] = (hidden(m, k) if case["fmt"] == "mx8" else normal(m, k) / math.sqrt(k)).to(TYPES[case["src"]])
    elif op == "norm":
        s["x"], s["residual"] = normal(m, k), hidden(m, k)
        s["gamma"], s["post_gamma"] = 0.3 * normal(k), 0.3 * normal(k)
        s["h"] = torch.empty(m, k, device=DEV)
    elif op == "gelu":
        s["gate_up"] = (1.5 * normal(m, 2 * k)).to(TYPES[case["src"]])
    else:
        n = case["n"]
        s["w"] = _planar(normal(n, k) / math.sqrt(k), "mx4")
        a = hidden(m, k)
        s["a"] = a if op == "linear" else a.bfloat16() if op == "rows" else _planar(a, case["fmt"])
        s["bias"] = normal(n) if case.get("bias") else None
        s["c"] = torch.empty(m, n, device=DEV, dtype=TYPES[case.get("out", "f32")])
    if op in ("quantize", "norm", "gelu"):
        bits = 8 if case["fmt"] == "mx8" else 4
        s["planar"] = torch.empty(m * k * bits // 8 + m * k // 32, device=DEV, dtype=torch.uint8)
        s["values"] = torch.empty(m, k, device=DEV, dtype=torch.bfloat16)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    m, k, op = case["m"], case["k"], case["op"]
    if op == "quantize":
        return _values(_planar(s["x"], case["fmt"]), case["fmt"], m, k).bfloat16()
    if op == "norm":
        u = s["x"]
        if case["post"]:
            u = u * (1.0 / torch.sqrt((u * u).mean(-1, keepdim=True) + EPS)) * (1.0 + s["post_gamma"])
        h = s["residual"] + u
        y = h * (1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)) * (1.0 + s["gamma"])
        return _values(_planar(y, case["fmt"]), case["fmt"], m, k).bfloat16(), h
    if op == "gelu":
        g, u = s["gate_up"][:, :k].float(), s["gate_up"][:, k:].float()
        inner = 2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)
        return _values(_planar(g / (1.0 + torch.exp(-inner)) * u, case["fmt"]), case["fmt"], m, k).bfloat16()
    a = _values(s["a"], case["fmt"], m, k) if op == "mx" else s["a"].float()
    c = a @ _values(s["w"], "mx4", case["n"], k).T
    if s["bias"] is not None:
        c = c + s["bias"]
    return c.to(s["c"].dtype)


def _run_own(s, case):
    rt = _package()
    m, k, op = case["m"], case["k"], case["op"]
    fmt = rt.MX_FP8 if case.get("fmt") == "mx8" else rt.MX_FP4
    if op == "quantize":
        rt.mx_quantize(s["x"], fmt, s["planar"], m, k)
    elif op == "norm":
        rt.add_rmsnorm_mx(s["x"], s["gamma"], EPS, fmt, s["planar"], m, k, residual=s["residual"],
                          post_gamma=s["post_gamma"] if case["post"] else None, sum_out=s["h"])
    elif op == "gelu":
        g = s["gate_up"]
        rt.gelu_mul_mx(g, g[:, k:], fmt, s["planar"], m, k, ld=2 * k)
    if op in ("quantize", "norm", "gelu"):
        rt.mx_dequantize(fmt, s["planar"], s["values"], m, k)
        return (s["values"], s["h"]) if op == "norm" else s["values"]
    n = case["n"]
    if op == "mx":
        rt.mx_gemm(fmt, s["a"], s["w"], s["c"], m, n, k, bias=s["bias"])
    elif op == "rows":
        rt.mxfp4_gemm(s["a"], s["w"], s["c"], m, n, k)
    elif m == 1 and s["bias"] is None:
        rt.mxfp4_gemv(s["w"], s["a"], s["c"], n, k)
    else:
        rt.qlinear_forward(rt.LINEAR_MXFP4, s["w"], s["a"], s["c"], m, n, k, bias=s["bias"])
    return s["c"]


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _times(x, e):
    """x 2^e in 64 bits, exactly."""
    return x * _power(e, 52, 1023, torch.int64, torch.float64)


def _grid(x, fmt):
    """The values that the microscaled form of x [rows][k] (float64) stands for: each block's exponent is that of its
    largest magnitude less the element's, each element a multiple of its own spacing, rounded half to even."""
    rows, k = x.shape
    b = x.reshape(rows, k // 32, 32)
    _, e = torch.frexp(b.abs().amax(-1, keepdim=True))          # |x| in [2^(e-1), 2^e)
    shared = torch.clamp(e - 1 - EMAX[fmt], min=-127)
    shared = torch.where(b.abs().amax(-1, keepdim=True) == 0, torch.full_like(shared, -127), shared)
    v = _times(b, -shared)
    mantissa, lowest = (3, -6) if fmt == "mx8" else (1, 0)
    _, ev = torch.frexp(v)
    spacing = torch.clamp(ev - 1, min=lowest) - mantissa
    q = _times(torch.round(_times(v, -spacing)), spacing).clamp(-LARGEST[fmt], LARGEST[fmt])
    return _times(q, shared).reshape(rows, k)


def _decode(planar, fmt, rows, k):
    """float64 values of a planar microscaled tensor, from the bits of sign, exponent and mantissa."""
    n = rows * k if fmt == "mx8" else rows * k // 2
    if fmt == "mx8":
        c = planar[:n].to(torch.int32)
        sign, e, f, bias, bits = c >> 7, (c >> 3) & 15, c & 7, 7, 3
    else:
        p = planar[:n].to(torch.int32)
        c = torch.stack([p & 15, p >> 4], -1).reshape(-1)
        sign, e, f, bias, bits = c >> 3, (c >> 1) & 3, c & 1, 1, 1
    whole = torch.where(e > 0, f + (1 << bits), f).double()
    v = _times(whole, torch.clamp(e, min=1) - bias - bits) * (1 - 2 * sign).double()
    x = planar[n:].to(torch.int32).reshape(-1, 1) - 127
    return _times(v.reshape(-1, 32), x).reshape(rows, k)


def exact(case, seed):
    s = prepare(case, seed)
    m, k, op = case["m"], case["k"], case["op"]
    if op == "quantize":
        return _grid(s["x"].double(), case["fmt"])
    if op == "norm":
        u = s["x"].double()
        if case["post"]:
            u = u / torch.sqrt(u.square().sum(-1, keepdim=True) / k + EPS) * (s["post_gamma"].double() + 1)
        h = u + s["residual"].double()
        y = h / torch.sqrt(h.square().sum(-1, keepdim=True) / k + EPS) * (s["gamma"].double() + 1)
        return _grid(y, case["fmt"]), h
    if op == "gelu":
        g, u = s["gate_up"][:, :k].double(), s["gate_up"][:, k:].double()
        y = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u
        return _grid(y, case["fmt"])
    a = _decode(s["a"], case["fmt"], m, k) if op == "mx" else s["a"].double()
    c = a @ _decode(s["w"], "mx4", case["n"], k).T
    return c if s["bias"] is None else c + s["bias"].double()
