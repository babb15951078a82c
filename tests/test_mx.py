"""The microscaled operators: rt_mx_quantize / rt_mx_dequantize, rt_add_rmsnorm_mx,
rt_gelu_mul_mx, and the products with an MXFP4 weight (rt_mx_gemm, rt_mxfp4_gemm,
rt_mxfp4_gemv, and the linear entry points with RT_LINEAR_MXFP4), against a plain
statement of the OCP MX formats in 64 bits.

The reference has none of these; parity with it is not at stake here."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

from conftest import rel_l2

FP4, FP8 = 4, 8
EMAX, TOP = {FP4: 2, FP8: 8}, {FP4: 6.0, FP8: 448.0}
E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], np.float64)


# ---------------------------------------------------------------------------
# the plain statement (float64, numpy)
# ---------------------------------------------------------------------------
def element(v, fmt):
    """v rounded to the nearest element, half to even, saturated."""
    mant, low = (3, -6) if fmt == FP8 else (1, 0)
    e = np.maximum(np.frexp(v)[1] - 1, low) - mant
    return np.clip(np.ldexp(np.round(np.ldexp(v, -e)), e), -TOP[fmt], TOP[fmt])


def scale_bytes(x, fmt):
    """e8m0 bytes of x [rows][k]: the exponent of each block's largest magnitude less the element's."""
    b = np.abs(x.reshape(x.shape[0], -1, 32))
    bad = ~np.isfinite(b).all(-1)
    top = np.where(np.isfinite(b), b, 0).max(-1)
    e = np.where(top > 0, np.frexp(top)[1] - 1, -1000)
    return np.where(bad, 255, np.maximum(e + 127 - EMAX[fmt], 0))


def values(x, fmt):
    """The values MX(x) stands for."""
    s = scale_bytes(x, fmt)[..., None]
    b = x.reshape(x.shape[0], -1, 32)
    with np.errstate(invalid="ignore"):
        q = np.ldexp(element(np.ldexp(b, 127 - s), fmt), s - 127)
    return np.where(s == 255, np.nan, q).reshape(x.shape)


def decode(buf, fmt, rows, k):
    """float64 values of a planar tensor's bytes."""
    n = rows * k if fmt == FP8 else rows * k // 2
    c, s = buf[:n].astype(np.int64), buf[n:n + rows * k // 32].astype(np.int64)
    if fmt == FP8:
        e, f = (c >> 3) & 15, c & 7
        v = np.where(e > 0, np.ldexp(8.0 + f, e - 10), np.ldexp(f.astype(np.float64), -9))
        v = np.where((c & 127) == 127, np.nan, v) * np.where(c >> 7, -1, 1)
    else:
        c = np.stack([c & 15, c >> 4], -1).reshape(-1)
        v = E2M1[c & 7] * np.where(c >> 3, -1, 1)
    sc = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    return (v.reshape(-1, 32) * sc[:, None]).reshape(rows, k)


def test_plain_statement_on_known_blocks():
    x = np.zeros((1, 32))
    x[0, :8] = [6, 5, 3.5, 2.5, 1.75, 0.75, 0.25, -0.3]  # scale 1 (byte 127): e2m1's own values and ties
    assert scale_bytes(x, FP4)[0, 0] == 127
    assert values(x, FP4)[0, :8].tolist() == [6, 4, 4, 2, 2, 1, 0, -0.5]
    x[0, 0] = 7.9  # the block's exponent stays that of 4: saturated
    assert values(x, FP4)[0, 0] == 6
    x[0, 0] = 8.0
    assert values(x, FP4)[0, 0] == 8 and scale_bytes(x, FP4)[0, 0] == 128
    x[0, 0] = 1.0
    assert scale_bytes(x, FP8)[0, 0] == 127 + 1 - 8 or x.max() != 1.0
    buf = np.zeros(33, np.uint8)
    buf[0], buf[1], buf[2], buf[32] = 0x7E, 0x01, 0xB8, 128
    assert decode(buf, FP8, 1, 32)[0, :3].tolist() == [896.0, 2.0 ** -8, -2.0]


# ---------------------------------------------------------------------------
# refusals (no GPU)
# ---------------------------------------------------------------------------
@pytest.fixture
def ptr():
    buf = (C.c_uint8 * 64)()
    p = (C.addressof(buf) + 15) & ~15
    p_keep = (p, buf)
    yield p_keep[0]


def refused(rt, status, word):
    assert status == rt.RT_EINVAL
    assert word in rt.lib().rt_last_error().decode()


def test_mx_bytes(rt):
    assert rt.mx_bytes(rt.MX_FP8, 3, 64) == 3 * 64 + 6
    assert rt.mx_bytes(rt.MX_FP4, 3, 64) == 3 * 32 + 6
    assert rt.mx_bytes(rt.MX_FP4, 3, 65) == 0 and rt.mx_bytes(5, 3, 64) == 0 and rt.mx_bytes(rt.MX_FP8, 0, 64) == 0
    assert rt.mx_bytes(rt.MX_FP8, 1 << 27, 1 << 10) == (1 << 37) + (1 << 32)
    assert rt.mx_bytes(rt.MX_FP8, 1 << 62, 1 << 10) == 0


def test_conversions_refuse_before_launch(rt, ptr):
    L = rt.lib()
    for call, last in ((lambda t, x, f, o, m, k: L.rt_mx_quantize(t, x, f, o, m, k, None), "x"),
                       (lambda t, x, f, o, m, k: L.rt_mx_dequantize(f, x, t, o, m, k, None), "src")):
        refused(rt, call(0, ptr, 5, ptr, 1, 32), "format 5")
        refused(rt, call(2, ptr, FP8, ptr, 1, 32), "type 2")
        refused(rt, call(0, ptr, FP8, ptr, 1, 48), "multiple of 32")
        refused(rt, call(0, ptr, FP8, ptr, 1, 0), "positive")
        refused(rt, call(0, ptr, FP8, ptr, -1, 32), "negative")
        refused(rt, call(0, ptr, FP8, ptr, 1 << 60, 1 << 30), "too large")
        refused(rt, call(0, None, FP8, ptr, 1, 32), "null")
        refused(rt, call(0, ptr, FP8, None, 1, 32), "null")
        refused(rt, call(1, ptr + 8, FP4, ptr, 1, 32), "aligned")
        refused(rt, call(1, ptr, FP4, ptr + 4, 1, 32), "aligned")
        assert call(0, None, FP4, None, 0, 32) == rt.RT_OK  # no rows: no work


def test_norm_refuses_before_launch(rt, ptr):
    L = rt.lib()

    def call(t=0, x=ptr, res=None, post=None, g=ptr, eps=1e-6, f=FP8, o=ptr, h=None, m=1, k=32):
        return L.rt_add_rmsnorm_mx(t, x, res, post, g, eps, f, o, h, m, k, None)

    refused(rt, call(f=3), "format 3")
    refused(rt, call(t=7), "type 7")
    refused(rt, call(k=40), "multiple of 32")
    refused(rt, call(k=32768 + 32), "exceeds")
    refused(rt, call(eps=-1.0), "eps")
    refused(rt, call(eps=float("nan")), "eps")
    refused(rt, call(x=None), "null")
    refused(rt, call(g=None), "null")
    refused(rt, call(o=None), "null")
    for name in ("x", "res", "post", "g", "o", "h"):
        refused(rt, call(**{name: ptr + 4}), "aligned")
    refused(rt, call(t=1, h=ptr), "bf16")
    assert call(m=0, x=None, g=None, o=None) == rt.RT_OK


def test_gelu_refuses_before_launch(rt, ptr):
    L = rt.lib()

    def call(t=0, g=ptr, u=ptr, ld=32, f=FP8, o=ptr, m=1, k=32):
        return L.rt_gelu_mul_mx(t, g, u, ld, f, o, m, k, None)

    refused(rt, call(f=0), "format 0")
    refused(rt, call(t=-1), "type -1")
    refused(rt, call(ld=28), "ld=28")
    refused(rt, call(ld=34), "ld=34")
    refused(rt, call(t=1, ld=36), "ld=36")  # whole 16 bytes are eight bf16
    refused(rt, call(k=33), "multiple of 32")
    refused(rt, call(g=None), "null")
    refused(rt, call(u=ptr + 4), "aligned")
    assert call(m=0) == rt.RT_OK


def test_products_refuse_before_launch(rt, ptr):
    L = rt.lib()
    calls = {
        "mx": lambda a=ptr, w=ptr, c=ptr, m=1, n=4, k=32: L.rt_mx_gemm(FP8, a, w, None, 0, c, m, n, k, None),
        "rows": lambda a=ptr, w=ptr, c=ptr, m=1, n=4, k=32: L.rt_mxfp4_gemm(0, a, w, c, m, n, k, None),
        "linear": lambda a=ptr, w=ptr, c=ptr, m=1, n=4, k=32: L.rt_qlinear_forward(rt.LINEAR_MXFP4, w, None, a, c, m, n, k, None),
        "gemm": lambda a=ptr, w=ptr, c=ptr, m=1, n=4, k=32: L.rt_linear_gemm_f32(rt.LINEAR_MXFP4, w, a, c, m, n, k, None),
        "batch": lambda a=ptr, w=ptr, c=ptr, m=1, n=4, k=32: L.rt_linear_gemv_batch(rt.LINEAR_MXFP4, w, a, c, m, n, k, None),
        "gemv": lambda a=ptr, w=ptr, c=ptr, m=1, n=4, k=32: L.rt_mxfp4_gemv(w, a, c, n, k, None),
    }
    for name, f in calls.items():
        refused(rt, f(k=48), "multiple of 32")
        refused(rt, f(n=0), "positive")
        refused(rt, f(k=-32), "positive")
        refused(rt, f(n=1 << 31), "int32")
        refused(rt, f(n=1 << 27), "too large")  # a grid's threads pass 2^32
        refused(rt, f(k=1 << 23), "too large")
        if name not in ("gemv", "batch"):
            refused(rt, f(m=1 << 30), "too large")
            refused(rt, f(m=1 << 20, n=1 << 16), "too large")
        for arg in ("a", "w", "c"):
            refused(rt, f(**{arg: None}), "null")
        for arg in ("a", "w"):
            refused(rt, f(**{arg: ptr + 4}), "aligned")
        if name != "gemv":
            assert f(m=0) == rt.RT_EINVAL and f(m=-1) == rt.RT_EINVAL
    assert calls["batch"](m=9) == rt.RT_EINVAL
    refused(rt, L.rt_mx_gemm(6, ptr, ptr, None, 0, ptr, 1, 4, 32, None), "format 6")
    refused(rt, L.rt_mx_gemm(FP4, ptr, ptr, None, 2, ptr, 1, 4, 32, None), "type 2")
    refused(rt, L.rt_mx_gemm(FP4, ptr, ptr, ptr + 2, 0, ptr, 1, 4, 32, None), "bias")
    refused(rt, L.rt_mx_gemm(FP4, ptr, ptr, None, 0, ptr + 2, 1, 4, 32, None), "aligned")
    refused(rt, L.rt_mx_gemm(FP4, ptr, ptr, None, 1, ptr + 1, 1, 4, 32, None), "aligned")
    refused(rt, L.rt_mxfp4_gemm(4, ptr, ptr, ptr, 1, 4, 32, None), "type 4")


@pytest.mark.parametrize("fmt", [0, 6, 7, 9])
def test_numbers_beside_the_formats_are_refused(rt, ptr, fmt):
    """A format number that names no format never reaches a kernel."""
    L = rt.lib()
    assert L.rt_linear_gemm_f32(fmt, ptr, ptr, ptr, 1, 16, 256, None) == rt.RT_EINVAL
    assert L.rt_qlinear_forward(fmt, ptr, None, ptr, ptr, 1, 16, 256, None) == rt.RT_EINVAL
    assert L.rt_linear_gemv_batch(fmt, ptr, ptr, ptr, 1, 16, 256, None) == rt.RT_EINVAL


def test_python_types(rt):
    import torch
    h = torch.zeros(32, dtype=torch.float16)
    f = torch.zeros(32)
    with pytest.raises(TypeError):
        rt.mx_quantize(h, rt.MX_FP8, f, 1, 32)
    with pytest.raises(TypeError):
        rt.gelu_mul_mx(f, f.bfloat16(), rt.MX_FP8, f, 1, 32)


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------
GUARD = 64


def out_bytes(rt, dev, fmt, rows, k):
    import torch
    return torch.full((rt.mx_bytes(fmt, rows, k) + GUARD,), 0xA5, dtype=torch.uint8, device=dev)


def fetch(buf, n):
    got = buf.cpu().numpy()
    assert np.all(got[n:] == 0xA5)  # what lies behind the tensor is left alone
    return got[:n]


def special_rows(k, seed):
    """Rows of f32: ordinary, tiny, huge, subnormal, ties of both formats, zeros, and blocks with inf and NaN."""
    rng = np.random.default_rng(seed)
    rows = [rng.normal(size=k), rng.normal(size=k) * 1e-30, rng.normal(size=k) * 2.0 ** 125,
            rng.normal(size=k) * 2.0 ** -140, np.ldexp(1.0, rng.integers(-149, 127, k)) * rng.choice([-1, 1], k),
            rng.choice(np.concatenate([E2M1, E2M1[:-1] + np.diff(E2M1) / 2, [5.0, 7.0, 7.5]]), k) * rng.choice([-1, 1], k),
            rng.integers(0, 256, k) * 2.0 + 1.0, np.zeros(k), rng.normal(size=k) * np.exp(3 * rng.normal(size=k))]
    x = np.array(rows).astype(np.float32)
    x[7, ::5] = -0.0
    bad = rng.normal(size=(2, k)).astype(np.float32)
    bad[0, 3], bad[1, k - 1] = np.inf, np.nan
    if k > 64:
        bad[0, 40] = -np.inf
    return np.concatenate([x, bad, np.full((1, k), np.finfo(np.float32).max, np.float32)])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [FP4, FP8])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("k", [32, 96, 1056, 8192])
def test_quantize_is_the_standard_conversion(rt, dev, fmt, bf16, k):
    import torch
    x = torch.from_numpy(special_rows(k, k)).to(dev)
    x = x.to(torch.bfloat16) if bf16 else x
    rows = x.shape[0]
    buf = out_bytes(rt, dev, fmt, rows, k)
    rt.mx_quantize(x, fmt, buf, rows, k)
    ref = x.float().cpu().numpy().astype(np.float64)
    got = fetch(buf, rt.mx_bytes(fmt, rows, k))
    n = rows * k * fmt // 8
    assert np.array_equal(got[n:].reshape(rows, -1), scale_bytes(ref, fmt))
    assert np.array_equal(decode(got, fmt, rows, k), values(ref, fmt), equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [FP4, FP8])
def test_dequantize_every_code_and_scale(rt, dev, fmt):
    import torch
    k = 512 if fmt == FP8 else 32  # all codes in a row; every scale byte on each of its blocks in turn
    codes = np.arange(256, dtype=np.uint8) if fmt == FP8 else (np.arange(16, dtype=np.uint8) | (np.arange(16, dtype=np.uint8)[::-1] << 4))
    codes = np.resize(codes, k * fmt // 8)
    rows = 256
    src = np.concatenate([np.tile(codes, rows), np.repeat(np.arange(256, dtype=np.uint8), k // 32)])
    ref = decode(src, fmt, rows, k)
    s = torch.from_numpy(src).to(dev)
    out = torch.full((rows * k + GUARD,), -7.0, device=dev)
    rt.mx_dequantize(fmt, s, out, rows, k)
    got = out.cpu().numpy()
    with np.errstate(over="ignore"):
        assert np.array_equal(got[:rows * k].reshape(rows, k), ref.astype(np.float32), equal_nan=True)
    assert np.all(got[rows * k:] == -7.0)
    half = torch.full((rows * k + GUARD,), -7.0, device=dev, dtype=torch.bfloat16)
    rt.mx_dequantize(fmt, s, half, rows, k)
    want = torch.from_numpy(ref).to(torch.float32).to(torch.bfloat16).float().numpy()
    got = half.float().cpu().numpy()
    assert np.array_equal(got[:rows * k].reshape(rows, k), want, equal_nan=True)
    assert np.all(got[rows * k:] == -7.0)


def within(got, y, fmt, tol):
    """got is MX of some y' with |y' - y| <= tol |y| (element by element, and for the block's scale)."""
    lo, hi = values(y * (1 - tol), fmt), values(y * (1 + tol), fmt)
    # a block whose largest value crosses a power of two between the two is rounded on either grid
    mid = values(y, fmt)
    least, most = np.minimum(np.minimum(lo, hi), mid), np.maximum(np.maximum(lo, hi), mid)
    bad = ~((got >= least) & (got <= most))
    return not np.any(bad & ~(np.isnan(got) & np.isnan(mid)))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [FP4, FP8])
@pytest.mark.parametrize("rows,k,post,res,bf16", [
    (1, 32, True, True, False), (1, 2560, True, True, False), (5, 1152, False, True, False), (7, 1056, True, False, True),
    (3, 96, False, False, False), (130, 2560, False, True, True), (2, 8192 + 32, True, True, False),
    (2, 16384 + 64, False, True, False), (1, 32768, True, True, True)])
def test_add_rmsnorm(rt, dev, fmt, rows, k, post, res, bf16):
    """h carries the rounding to f32 alone (2^-24) and y two: h / rms(h) (1 + gamma) in 64 bits, to f32, to the element."""
    import torch
    rng = np.random.default_rng(rows + k)
    x = rng.normal(size=(rows, k)).astype(np.float32)
    x[:, 7] *= 1000
    r = (rng.normal(size=(rows, k)) * np.exp(rng.normal(size=(rows, 1)))).astype(np.float32)
    if rows > 2:
        x[1], r[1] = 0, 0  # a row of zeros: eps alone keeps it finite
    xt = torch.from_numpy(x).to(dev)
    xt = xt.to(torch.bfloat16) if bf16 else xt
    g, pg = (0.3 * rng.normal(size=k)).astype(np.float32), (0.3 * rng.normal(size=k)).astype(np.float32)
    gt, pt, rtt = (torch.from_numpy(v).to(dev) for v in (g, pg, r))
    eps = float(np.float32(1e-6))
    u = xt.float().cpu().numpy().astype(np.float64)
    if post:
        u = u / np.sqrt((u * u).mean(-1, keepdims=True) + eps) * (1 + pg.astype(np.float64))
    h = u + (r.astype(np.float64) if res else 0)
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * (1 + g.astype(np.float64))
    buf = out_bytes(rt, dev, fmt, rows, k)
    ho = torch.full((rows * k + GUARD,), -7.0, device=dev)
    args = dict(residual=rtt if res else None, post_gamma=pt if post else None)
    rt.add_rmsnorm_mx(xt, gt, eps, fmt, buf, rows, k, sum_out=ho, **args)
    hg = ho.cpu().numpy()
    assert np.all(hg[rows * k:] == -7.0)
    # 64-bit sums of up to 32768 terms are off by far less than 2^-30
    assert np.all(np.abs(hg[:rows * k].reshape(rows, k) - h) <= np.abs(h) * (2.0 ** -24 + 2.0 ** -30) + 1e-40
                  + (np.abs(u) + np.abs(r)) * 2.0 ** -40)
    got = fetch(buf, rt.mx_bytes(fmt, rows, k))
    assert within(decode(got, fmt, rows, k), y, fmt, 2.0 ** -23)
    # without sum_out the same codes; in place (over the residual, over x) too
    again = out_bytes(rt, dev, fmt, rows, k)
    rt.add_rmsnorm_mx(xt, gt, eps, fmt, again, rows, k, **args)
    assert np.array_equal(fetch(again, got.size), got)
    for over in ((["residual"] if res else []) + ([] if bf16 else ["x"])):
        a = dict(args)
        xx = xt.clone()
        if res:
            a["residual"] = rtt.clone()
        rt.add_rmsnorm_mx(xx, gt, eps, fmt, again, rows, k, sum_out=xx if over == "x" else a["residual"], **a)
        assert np.array_equal(fetch(again, got.size), got)
        assert np.array_equal((xx if over == "x" else a["residual"]).cpu().numpy().reshape(-1), hg[:rows * k])


@pytest.mark.gpu
def test_add_rmsnorm_keeps_bad_rows_apart(rt, dev):
    import torch
    rows, k = 4, 64
    x = np.random.default_rng(2).normal(size=(rows, k)).astype(np.float32)
    x[1, 5], x[2, 40] = np.nan, np.inf
    buf = out_bytes(rt, dev, FP8, rows, k)
    ho = torch.empty(rows, k, device=dev)
    rt.add_rmsnorm_mx(torch.from_numpy(x).to(dev), torch.zeros(k, device=dev), 1e-6, FP8, buf, rows, k, sum_out=ho)
    got = decode(fetch(buf, rt.mx_bytes(FP8, rows, k)), FP8, rows, k)
    assert np.all(np.isnan(got[1])) and np.all(np.isfinite(got[[0, 3]]))
    assert np.all(np.isnan(got[2, 32:])) and np.all(got[2, :32] == 0)  # finite / inf is 0, inf / inf NaN
    assert np.array_equal(ho.cpu().numpy(), x, equal_nan=True)


def gelu64(v):
    return 0.5 * v * (1 + np.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [FP4, FP8])
@pytest.mark.parametrize("rows,k,bf16,fused", [(1, 32, False, False), (5, 6912, False, True), (33, 1056, True, True),
                                               (300, 96, True, False), (3, 10240, False, False)])
def test_gelu_mul(rt, dev, fmt, rows, k, bf16, fused):
    """y = g / (1 + 2^z) u, |z| <= 2.31 |g| (1 + 0.045 g^2): z has three roundings of 2^-24 |z|, its power 0.7 of that
    and 2^-23 more, the quotient, its product with g and that with u 2^-23, 2^-24 and 2^-24."""
    import torch
    rng = np.random.default_rng(rows + k)
    gu = (1.5 * rng.normal(size=(rows, 2 * k))).astype(np.float32)
    t = torch.from_numpy(gu).to(dev)
    t = t.to(torch.bfloat16) if bf16 else t
    gu = t.float().cpu().numpy().astype(np.float64)
    g, u = gu[:, :k], gu[:, k:]
    with np.errstate(all="ignore"):
        z = 2.31 * np.abs(g) * (1 + 0.045 * g * g)
    tol = (6 + 2.1 * z) * 2.0 ** -24
    buf = out_bytes(rt, dev, fmt, rows, k)
    if fused:
        rt.gelu_mul_mx(t, t[:, k:], fmt, buf, rows, k, ld=2 * k)
    else:
        rt.gelu_mul_mx(t[:, :k].contiguous(), t[:, k:].contiguous(), fmt, buf, rows, k)
    got = decode(fetch(buf, rt.mx_bytes(fmt, rows, k)), fmt, rows, k)
    assert within(got, gelu64(g) * u, fmt, tol)


@pytest.mark.gpu
def test_gelu_mul_extremes(rt, dev):
    """Large |gate| gives gate or zero, an infinity or NaN its own block alone."""
    import torch
    g = np.zeros((1, 160), np.float32)
    g[0, :8] = [1e30, -1e30, 88.0, -88.0, 12.0, -12.0, 3e38, -3e38]
    g[0, 32:36] = [1e-30, -1e-30, 1e-40, -1e-42]
    g[0, 64], g[0, 96] = np.nan, np.inf
    g[0, 128] = 5.0
    u = np.ones((1, 160), np.float32)
    buf = out_bytes(rt, dev, FP8, 1, 160)
    rt.gelu_mul_mx(torch.from_numpy(g).to(dev), torch.from_numpy(u).to(dev), FP8, buf, 1, 160)
    got = decode(fetch(buf, rt.mx_bytes(FP8, 1, 160)), FP8, 1, 160)[0]
    want = values(np.where(g[:, :32] > 20, g[:, :32], 0).astype(np.float64), FP8)[0]
    assert np.array_equal(got[:32], want)
    assert np.array_equal(got[32:64], values(g[:, 32:64].astype(np.float64) * 0.5, FP8)[0])
    assert np.all(np.isnan(got[64:128])) and np.all(np.isfinite(got[128:])) and got[128] == 5.0


# --- products -------------------------------------------------------------
def planar(x, fmt):
    """MX(x) as planar bytes, from the plain statement."""
    s = scale_bytes(x, fmt)
    v = np.ldexp(x.reshape(x.shape[0], -1, 32), 127 - s[..., None])
    q = element(v, fmt).reshape(-1)
    a, sign = np.abs(q), (np.signbit(q)).astype(np.uint8)
    if fmt == FP8:
        e = np.maximum(np.frexp(a)[1] - 1, -6)
        m = np.ldexp(a, 3 - e).astype(np.int64)  # 0..15
        code = np.where(m >= 8, ((e + 7) << 3) | (m - 8), m).astype(np.uint8) | (sign << 7)
    else:
        code = np.searchsorted(E2M1, a).astype(np.uint8) | (sign << 3)
        code = code[0::2] | (code[1::2] << 4)
    return np.concatenate([code.astype(np.uint8), s.reshape(-1).astype(np.uint8)])


def test_planar_statement_round_trips():
    x = np.random.default_rng(0).normal(size=(5, 96))
    for fmt in (FP4, FP8):
        assert np.array_equal(decode(planar(x, fmt), fmt, 5, 96), values(x, fmt))


PLANES = {"f32": 5, "bf16": 3, FP8: 2, FP4: 1}
FLOOR = {"f32": 2.0 ** -30, "bf16": 2.0 ** -20}  # of a block's largest value: what a digit form drops


def product(rt, dev, act, a, w, m, n, k, bias=None, out="f32", call="gemm", stream=None):
    """One product; a and w are device tensors.  Returns [m][n] float64 after checking what lies behind c."""
    import torch
    c = torch.full((m * n + GUARD,), -7.0, device=dev, dtype=torch.float32 if out == "f32" else torch.bfloat16)
    if act in (FP4, FP8):
        rt.mx_gemm(act, a, w, c, m, n, k, bias=bias, stream=stream)
    elif call == "linear":
        rt.qlinear_forward(rt.LINEAR_MXFP4, w, a, c, m, n, k, bias=bias, stream=stream)
    elif call == "batch":
        rt.linear_gemv_batch(rt.LINEAR_MXFP4, w, a, c, m, n, k, stream=stream)
    elif call == "gemv":
        rt.mxfp4_gemv(w, a, c, n, k, stream=stream)
    else:
        rt.mxfp4_gemm(a, w, c, m, n, k, stream=stream)
    torch.cuda.synchronize()
    got = c.double().cpu().numpy()
    assert np.all(got[m * n:] == -7.0)
    return got[:m * n].reshape(m, n)


def make(dev, act, m, n, k, seed, spread=0.0):
    """Activations and weight as device tensors and as float64."""
    import torch
    rng = np.random.default_rng(seed)
    a = rng.normal(size=(m, k)) * np.exp(spread * rng.normal(size=(m, k)))
    w = planar(rng.normal(size=(n, k)) / math.sqrt(k), FP4)
    w64 = decode(w, FP4, n, k)
    if act in (FP4, FP8):
        p = planar(a, act)
        return torch.from_numpy(p).to(dev), torch.from_numpy(w).to(dev), decode(p, act, m, k), w64
    t = torch.from_numpy(a.astype(np.float32))
    t = t.to(torch.bfloat16) if act == "bf16" else t
    return t.to(dev), torch.from_numpy(w).to(dev), t.double().numpy(), w64


def check(got, a64, w64, act, k, bias=None, out="f32"):
    """Products of 4-bit weights with e2m1, e4m3 (in two halves) or a plane's digits are exact.  An instruction adds 16
    group sums and the accumulator, each cut at 2^-25 of the largest and the sum rounded: 9 times 2^-24 per 128 of K
    and plane; one rounding for each of up to 64 K splits and one of the bias.  A digit form is off by 2^-24 of the
    value and FLOOR of its block's largest.  MXFP8 into bf16 is one instruction: each of eight neighbouring products
    is cut at 2^-13 of the largest exponent sum among them."""
    if not got.size:
        return
    ref, mag = a64 @ w64.T, np.abs(a64) @ np.abs(w64).T
    tol = mag * (9 * PLANES[act] * -(-k // 128) + 65) * 2.0 ** -24
    if act in FLOOR:
        blocks = np.abs(a64).reshape(a64.shape[0], -1, 32).max(-1)
        tol = tol + np.repeat(blocks, 32, -1) @ np.abs(w64).T * FLOOR[act]
    if bias is not None:
        ref = ref + bias
        tol = tol + np.abs(bias) * 2.0 ** -23
    if out == "bf16":
        if act == FP8:
            ga, gw = (np.abs(v).reshape(v.shape[0], -1, 8).max(-1) for v in (a64, w64))
            tol = tol + 8 * 2.0 ** -13 * (ga @ gw.T)
            # every element's rounding is at most 2^-8 of it, so the norm's is too; the cuts are signed, the largest
            # 2^-13 of a term: together below 2^-12 of the result's norm
            assert np.linalg.norm(got - ref) < (2.0 ** -8 + 2.0 ** -12) * np.linalg.norm(ref)
        tol = tol + np.abs(ref) * 2.0 ** -8
    assert np.all(np.abs(got - ref) <= tol + 1e-37)


SHAPES = [(1, 1, 32), (1, 17, 96), (1, 300, 2560), (2, 33, 160), (3, 130, 1152), (4, 16, 128), (5, 257, 6912),
          (8, 100, 4128), (15, 31, 64), (17, 65, 544), (33, 129, 1056), (64, 128, 512), (65, 64, 1024), (100, 515, 736),
          (128, 256, 256), (129, 300, 1184), (257, 130, 2560), (300, 1025, 416)]


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16", FP8, FP4])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_matches_float64(rt, dev, act, m, n, k):
    import torch
    a, w, a64, w64 = make(dev, act, m, n, k, m + n + k)
    got = product(rt, dev, act, a, w, m, n, k)
    check(got, a64, w64, act, k)
    assert np.array_equal(got, product(rt, dev, act, a, w, m, n, k))  # the order of the sum is fixed
    bias = np.random.default_rng(1).normal(size=n).astype(np.float32)
    bt = torch.from_numpy(bias).to(dev)
    if act == "f32":
        check(product(rt, dev, act, a, w, m, n, k, bias=bt, call="linear"), a64, w64, act, k, bias.astype(np.float64))
        if m <= 8:
            check(product(rt, dev, act, a, w, m, n, k, call="batch"), a64, w64, act, k)
        if m == 1:
            check(product(rt, dev, act, a, w, m, n, k, call="gemv"), a64, w64, act, k)
    elif act != "bf16":
        check(product(rt, dev, act, a, w, m, n, k, bias=bt, out="bf16"), a64, w64, act, k, bias.astype(np.float64), "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("act,m,n,k,out", [(FP4, 4090, 4100, 32, "f32"), (FP4, 4096, 4104, 256, "bf16"), (FP4, 4000, 4097, 288, "bf16"),
                                           (FP4, 4001, 4352, 640, "f32"), (FP4, 3841, 4088, 1056, "bf16"), (FP8, 4090, 4100, 160, "bf16"),
                                           (FP8, 3900, 4097, 544, "f32"), ("f32", 3841, 4100, 96, "f32"), ("bf16", 4000, 4096, 416, "f32")])
def test_products_of_many_tiles(rt, dev, act, m, n, k, out):
    """Sizes that fill every CU with whole tiles, their last rows, columns and pieces of K ragged."""
    a, w, a64, w64 = make(dev, act, m, n, k, 21)
    check(product(rt, dev, act, a, w, m, n, k, out=out), a64, w64, act, k, out=out)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 6, 40, 200])
def test_f32_activations_keep_their_bits(rt, dev, m):
    """Activations over 2^+-12 within a block, and rows at 2^90 and 2^-90, against the exact product."""
    import torch
    n, k = 70, 640
    a, w, a64, w64 = make(dev, "f32", m, n, k, 5, spread=3.0)
    a64 = a64 * np.where(np.arange(m) % 3 == 1, 2.0 ** 90, np.where(np.arange(m) % 3 == 2, 2.0 ** -90, 1.0))[:, None]
    a64[m // 2, 64:96] = 0
    check(product(rt, dev, "f32", torch.from_numpy(a64.astype(np.float32)).to(dev), w, m, n, k), a64, w64, "f32", k)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16", FP8, FP4])
@pytest.mark.parametrize("m", [1, 5, 37, 150])
def test_bad_values_stay_in_their_rows_and_columns(rt, dev, act, m):
    """A NaN or infinity among the activations gives a row of NaN, a scale of 255 in the weight a column."""
    import torch
    n, k = 150, 288
    a, w, a64, w64 = make(dev, act, m, n, k, 9)
    row = m // 2
    if act in (FP4, FP8):
        a = a.clone()
        a[m * k * act // 8 + row * (k // 32) + 8] = 255  # the row's last block
    else:
        a = a.clone()
        a[row, k - 1] = math.inf if m == 5 else math.nan
    got = product(rt, dev, act, a, w, m, n, k)
    assert np.all(np.isnan(got[row]))
    keep = np.arange(m) != row
    check(got[keep], a64[keep], w64, act, k)
    w = w.clone()
    w[n * k // 2 + 77 * (k // 32) + 8] = 255
    got = product(rt, dev, act, a, w, m, n, k)
    cols = np.arange(n) != 77
    assert np.all(np.isnan(got[:, 77]))
    check(got[keep][:, cols], a64[keep], w64[cols], act, k)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", FP8, FP4])
@pytest.mark.parametrize("m", [1, 9, 130])
def test_ends_of_the_scale_range(rt, dev, act, m):
    """Weight scales 2^-127 and 2^120 beside ordinary ones, zero weights and zero activations."""
    import torch
    n, k = 20, 256
    a, w, a64, w64 = make(dev, act, m, n, k, 11)
    wh = w.cpu().numpy().copy()
    s = wh[n * k // 2:].reshape(n, k // 32)
    s[3], s[4], s[5, ::2] = 0, 247 - 10, 240
    wh[6 * k // 2:7 * k // 2] = 0
    w64 = decode(wh, FP4, n, k)
    got = product(rt, dev, act, a, torch.from_numpy(wh).to(dev), m, n, k)
    check(got, a64, w64, act, k)
    assert np.all(got[:, 6] == 0)


@pytest.mark.gpu
def test_offsets_past_32_bits(rt, dev):
    """A bf16 tensor of 2^32 + 2^16 elements (8 GiB in), and a weight whose codes pass 2^32 bytes: the far ends."""
    import torch
    k = 1 << 16
    rows = (1 << 16) + 1
    x = torch.zeros(rows * k, dtype=torch.bfloat16, device=dev)
    x[-k:] = torch.randn(k, device=dev).to(torch.bfloat16)
    buf = torch.full((rt.mx_bytes(FP4, rows, k) + GUARD,), 0xA5, dtype=torch.uint8, device=dev)
    rt.mx_quantize(x, FP4, buf, rows, k)
    last = x[-k:].float().cpu().numpy().astype(np.float64)[None]
    del x
    n = rows * k // 2
    got = np.concatenate([buf[n - k // 2:n].cpu().numpy(), buf[n + (rows - 1) * (k // 32):n + rows * (k // 32)].cpu().numpy()])
    assert np.array_equal(decode(got, FP4, 1, k), values(last, FP4))
    assert bool((buf[-GUARD:] == 0xA5).all()) and int(buf[:n - k // 2].max()) == 0
    del buf
    n, k = (1 << 17) + 40, 1 << 16
    w = torch.zeros(rt.mx_bytes(FP4, n, k), dtype=torch.uint8, device=dev)
    tail = planar(np.random.default_rng(3).normal(size=(40, k)), FP4)
    w[(n - 40) * k // 2:n * k // 2] = torch.from_numpy(tail[:40 * k // 2]).to(dev)
    w[-40 * k // 32:] = torch.from_numpy(tail[40 * k // 2:]).to(dev)
    for m in (1, 20):
        a = torch.randn(m, k, device=dev)
        c = torch.full((m, n), -7.0, device=dev)
        rt.mxfp4_gemm(a, w, c, m, n, k)
        check(c[:, -40:].double().cpu().numpy(), a.double().cpu().numpy(), decode(tail, FP4, 40, k), "f32", k)
        assert bool((c[:, :-40] == 0).all())


@pytest.mark.gpu
def test_feed_forward_in_microscaled_steps(rt, dev):
    """residual + norm -> gate|up -> gated GELU -> down, as a layer runs them, each step against its plain form on the
    same inputs, and the whole against 64 bits without any rounding."""
    import torch
    m, h, f = 37, 512, 1056
    rng = np.random.default_rng(8)
    x, res = (torch.from_numpy(rng.normal(size=(m, h)).astype(np.float32)).to(dev) for _ in range(2))
    g, pg = (torch.from_numpy((0.2 * rng.normal(size=h)).astype(np.float32)).to(dev) for _ in range(2))
    wgu = rng.normal(size=(2 * f, h)).astype(np.float32) / math.sqrt(h)
    wd = rng.normal(size=(h, f)).astype(np.float32) / math.sqrt(f)

    def weight(w):
        buf = torch.empty(rt.mx_bytes(FP4, *w.shape), dtype=torch.uint8, device=dev)
        rt.mx_quantize(torch.from_numpy(w).to(dev), FP4, buf, *w.shape)
        return buf, decode(buf.cpu().numpy(), FP4, *w.shape)

    (wgu_d, wgu64), (wd_d, wd64) = weight(wgu), weight(wd)
    hs = torch.empty(m, h, device=dev)
    a = torch.empty(rt.mx_bytes(FP8, m, h), dtype=torch.uint8, device=dev)
    gu = torch.empty(m, 2 * f, device=dev, dtype=torch.bfloat16)
    b = torch.empty(rt.mx_bytes(FP8, m, f), dtype=torch.uint8, device=dev)
    y = torch.empty(m, h, device=dev)
    rt.add_rmsnorm_mx(x, g, 1e-6, FP8, a, m, h, residual=res, post_gamma=pg, sum_out=hs)
    rt.mx_gemm(FP8, a, wgu_d, gu, m, 2 * f, h)
    rt.gelu_mul_mx(gu, gu[:, f:], FP8, b, m, f, ld=2 * f)
    rt.mx_gemm(FP8, b, wd_d, y, m, h, f)
    torch.cuda.synchronize()
    a64, b64 = decode(a.cpu().numpy(), FP8, m, h), decode(b.cpu().numpy(), FP8, m, f)
    gu64 = gu.double().cpu().numpy()
    check(gu64, a64, wgu64, FP8, h, out="bf16")
    check(y.double().cpu().numpy(), b64, wd64, FP8, f)
    u = x.double().cpu().numpy()
    u = u / np.sqrt((u * u).mean(-1, keepdims=True) + 1e-6) * (1 + pg.double().cpu().numpy())
    hh = u + res.double().cpu().numpy()
    n = hh / np.sqrt((hh * hh).mean(-1, keepdims=True) + 1e-6) * (1 + g.double().cpu().numpy())
    p = n @ wgu64.T
    ref = (gelu64(p[:, :f]) * p[:, f:]) @ wd64.T
    got = y.double().cpu().numpy()
    # two e4m3 roundings of 2^-4 at most (uniform: 2^-4 / sqrt(3) of a value near its power of two, less above),
    # independent over the terms of a sum; the gate's error enters the product twice at most
    assert np.linalg.norm(got - ref) / np.linalg.norm(ref) < 3 * 2.0 ** -4 / math.sqrt(3)


@pytest.mark.gpu
def test_graph_replays_and_other_streams(rt, dev):
    """A captured norm -> product -> GELU -> product chain, replayed with eager work of other sizes in between, and
    the same chain on a stream of its own: always the eager result."""
    import torch
    m, h, f = 20, 256, 512

    def state(seed):
        rng = np.random.default_rng(seed)
        t = lambda *s: torch.from_numpy(rng.normal(size=s).astype(np.float32)).to(dev)  # noqa: E731
        s = dict(x=t(m, h), res=t(m, h), g=t(h), a=torch.empty(rt.mx_bytes(FP8, m, h), dtype=torch.uint8, device=dev),
                 gu=torch.empty(m, 2 * f, device=dev), b=torch.empty(rt.mx_bytes(FP4, m, f), dtype=torch.uint8, device=dev),
                 y=torch.empty(m, h, device=dev), z=torch.empty(m, 300, device=dev))
        for name, n, k in (("w1", 2 * f, h), ("w2", h, f), ("w3", 300, h)):
            s[name] = torch.from_numpy(planar(rng.normal(size=(n, k)) / math.sqrt(k), FP4)).to(dev)
        return s

    def chain(s, stream=None):
        rt.add_rmsnorm_mx(s["x"], s["g"], 1e-6, FP8, s["a"], m, h, residual=s["res"], stream=stream)
        rt.mx_gemm(FP8, s["a"], s["w1"], s["gu"], m, 2 * f, h, stream=stream)
        rt.gelu_mul_mx(s["gu"], s["gu"][:, f:], FP4, s["b"], m, f, ld=2 * f, stream=stream)
        rt.mx_gemm(FP4, s["b"], s["w2"], s["y"], m, h, f, stream=stream)
        rt.mxfp4_gemm(s["y"], s["w3"], s["z"], m, 300, h, stream=stream)

    s = state(1)
    chain(s)
    torch.cuda.synchronize()
    want = [s[k].clone() for k in ("gu", "y", "z")]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(s, side)  # the workspace of this stream grows outside the capture
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        chain(s, side)
    other = state(2)
    for i in range(4):
        for k in ("gu", "y", "z"):
            s[k].zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s[k], w) for k, w in zip(("gu", "y", "z"), want)), i
        chain(other)
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_capture_that_would_allocate_is_refused(rt, dev):
    """A captured call whose workspace does not exist yet fails with RT_ESTATE; the same call runs afterwards."""
    import torch
    m, n, k = 64, 64, 4096
    a, w = torch.randn(m, k, device=dev), torch.zeros(rt.mx_bytes(FP4, n, k), dtype=torch.uint8, device=dev)
    c = torch.empty(m, n, device=dev)
    s = torch.cuda.Stream()
    rt.gemm_workspace_release(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    seen = None
    with torch.cuda.graph(graph, stream=s):
        try:
            rt.mxfp4_gemm(a, w, c, m, n, k, stream=s)
        except rt.RtError as e:
            seen = e
    assert seen is not None and seen.code == rt.RT_ESTATE
    rt.mxfp4_gemm(a, w, c, m, n, k, stream=s)
    s.synchronize()
    assert bool((c == 0).all()) and rt.gemm_workspace_held(s) > 0
    rt.gemm_workspace_release(s)


# --- the decode engine with MXFP4 projections -------------------------------
PROJ = ("q", "k", "v", "o", "gate", "up", "down")
MX, Q8_0, BF16, Q6K = 8, 5, 2, 4
ENGINE = {  # layer -> projection -> format, Q4_K otherwise
    # every set by itself, behind Q4_K sets, and beside each other format
    "tiny": {0: {p: MX for p in PROJ}, 1: dict(v=MX, down=MX), 2: dict(q=MX, up=MX), 3: dict(q=Q8_0, k=MX, v=BF16, o=MX),
             4: dict(q=MX, k=Q6K, v=MX, gate=Q8_0, up=MX), 5: {p: MX for p in PROJ}},
    "768": {0: {p: MX for p in PROJ}, 1: dict(v=MX, gate=MX, down=MX), 2: dict(q=MX, k=Q8_0, v=MX, o=MX, up=MX)},
    "1152": {0: dict({p: Q8_0 for p in PROJ}, v=MX, o=MX, down=MX), 1: {p: MX for p in PROJ}},
}


def engine_cfg(shape):
    if shape == "tiny":
        from test_gpu_decode import tiny
        return tiny(2)
    hidden, ffn, heads, dim = dict(zip(("768", "1152"), ((768, 1536, 4, 128), (1152, 6912, 4, 256))))[shape]
    return dict(hidden=hidden, ffn=ffn, n_q_heads=heads, n_kv_heads=1, head_dim=dim, n_layers=len(ENGINE[shape]), vocab=777,
                sliding_window=9, global_every=2, rope_theta_local=10000.0, rope_theta_global=1000000.0,
                rope_fs_local=1.0, rope_fs_global=0.125, eps=1e-6, attn_scale=1.0 / math.sqrt(dim))


def engine_model(orc, shape, max_seq, ctx, seed):
    """The oracle's layers hold an MXFP4 projection's values as bf16, which has
    every one of them (2 significant bits); the device's hold its bytes."""
    from test_kquant import SHAPES, apply_formats
    from test_oracle import make_model
    cfg, plan = engine_cfg(shape), ENGINE[shape]
    if cfg["hidden"] % 256:  # no Q4_K blocks: make_model's weights are replaced by the plan's, which has every projection
        layers, embed, fnorm = make_model_any(orc, cfg, max_seq, ctx, seed)
    else:
        layers, embed, fnorm = make_model(orc, cfg, max_seq=max_seq, ctx=ctx, seed=seed)
    as_bf16 = {li: {p: BF16 if f == MX else f for p, f in d.items()} for li, d in plan.items()}
    dev_layers, fmts = apply_formats(orc, cfg, layers, as_bf16, seed=seed + 1)
    for li, d in plan.items():
        for p, f in d.items():
            if f != MX:
                continue
            x = (layers[li][p].astype(np.uint32) << 16).view(np.float32).astype(np.float64).reshape(SHAPES(cfg)[p])
            dev_layers[li][p] = planar(x, FP4)
            v = values(x, FP4).astype(np.float32).reshape(-1)
            layers[li][p] = (v.view(np.uint32) >> 16).astype(np.uint16)
            assert np.array_equal((layers[li][p].astype(np.uint32) << 16).view(np.float32), v)
            fmts[li][PROJ.index(p)] = MX
    return cfg, layers, dev_layers, fmts, embed, fnorm


def make_model_any(orc, cfg, max_seq, ctx, seed):
    rng = np.random.default_rng(seed)
    H, D, KVD = cfg["hidden"], cfg["head_dim"], cfg["n_kv_heads"] * cfg["head_dim"]
    layers = []
    for _ in range(cfg["n_layers"]):
        L = {n: (0.1 * rng.normal(size=s)).astype(np.float32) for n, s in
             dict(in_norm=H, post_attn_norm=H, pre_ffn_norm=H, post_ffn_norm=H, q_norm=D, k_norm=D).items()}
        for c in ("k_cache", "v_cache"):
            L[c] = np.zeros((max_seq, KVD), np.float32)
            L[c][:ctx] = rng.normal(size=(ctx, KVD))
        layers.append(L)
    return layers, orc.synth_bf16(seed, cfg["vocab"] * H), (0.1 * rng.normal(size=H)).astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", ENGINE)
def test_engine_steps_and_verify_batch(rt, orc, shape):
    """Steps (one eager, the others replays), then batches of 3 and of 8, against
    the oracle on the same values.  Tolerance: the engine's for every format."""
    from test_kquant import mixed_ctx
    ctx, max_seq = 6, 40
    cfg, layers, dev_layers, fmts, embed, fnorm = engine_model(orc, shape, max_seq, ctx, 9000)
    d = mixed_ctx(rt, cfg, dev_layers, fmts, embed, fnorm, ctx, max_seq, layers)
    assert d.verify_batched
    for tok in (11, 3, 700):
        got = d.decode_step(tok, ctx)
        ref = orc.gemma3_decode_step(cfg, layers, embed, fnorm, token=tok, pos=ctx)
        print(f"step {ctx}: {rel_l2(got, ref):.2e}", flush=True)
        assert rel_l2(got, ref) < 1e-3, (ctx, rel_l2(got, ref))
        ctx += 1
    for m in (3, 8):
        toks = [(31 * i + m) % cfg["vocab"] for i in range(m)]
        for _ in range(2):  # the second is a replay
            got = d.decode_step_batch(toks, ctx)
        for i, tok in enumerate(toks):
            ref = orc.gemma3_decode_step(cfg, layers, embed, fnorm, token=tok, pos=ctx + i)
            print(f"batch {m} row {i}: {rel_l2(got[i], ref):.2e}", flush=True)
            assert rel_l2(got[i], ref) < 1e-3, (m, i, rel_l2(got[i], ref))
        ctx += m
    d.close()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,T,mode,chunk", [("tiny", 3, 1, 0), ("tiny", 20, 0, 0), ("768", 37, 1, 0), ("1152", 30, 1, 7)])
def test_engine_prefill(rt, orc, shape, T, mode, chunk):
    """Prompts through the GEMM on widened rows and, in chunks of 7, through the
    batched products; the step after a prompt reads its cache."""
    from test_kquant import plain_ctx
    from test_prefill import LOGITS_TOL, fresh_caches
    cfg, layers, dev_layers, fmts, embed, fnorm = engine_model(orc, shape, 48, 0, 9100 + T)
    d = plain_ctx(rt, cfg, dev_layers, fmts, embed, fnorm, 48)
    if chunk:
        d.set_prefill_chunk(chunk)
    toks = [(17 * i + 4) % cfg["vocab"] for i in range(T)]
    got = d.prefill(toks, 0, mode)
    ref_layers = fresh_caches(layers)
    ref = orc.gemma3_prefill(cfg, ref_layers, embed, fnorm, toks, 0, mode)
    print(f"prefill: {rel_l2(got, ref):.2e}", flush=True)
    assert rel_l2(got, ref) < LOGITS_TOL, rel_l2(got, ref)
    if mode == 1:
        ref = orc.gemma3_decode_step(cfg, ref_layers, embed, fnorm, token=9, pos=T)
        assert rel_l2(d.decode_step(9, T), ref) < LOGITS_TOL
    d.close()
