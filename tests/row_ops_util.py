"""The row operators in 64 bits (layer norm, dropout with a regenerated mask, residual norm) and the error bounds their
fp32 kernels are held to.  Written from the definitions; gradients come from double-precision automatic differentiation
of the forward definition, not from the kernels' formulas."""
import math

import numpy as np
import torch

U = 2.0 ** -24          # half a step of fp32, relative
CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def philox4x32_10(c, k):
    """Philox4x32-10 (Salmon et al., SC'11) on arrays of counters [..., 4] with one key (k0, k1)."""
    c = [np.asarray(v, np.uint64) for v in c]
    m = np.uint64(0xFFFFFFFF)
    k0, k1 = k
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def draws(rows, width, seed, step=0, layer=0, row_offset=0):
    """u(i, j), [rows, width]."""
    out = np.zeros((rows, -(-width // 8), 8), np.int64)
    row = np.arange(rows, dtype=np.uint64)[:, None] + np.uint64(row_offset)
    unit = np.arange(out.shape[1], dtype=np.uint64)[None, :]
    zero = row * np.uint64(0) + unit * np.uint64(0)
    words = philox4x32_10([(row & np.uint64(0xFFFFFFFF)) + zero, unit | ((row >> np.uint64(32)) << np.uint64(21)),
                           zero + np.uint64(layer | 1 << 31), zero + np.uint64(step & 0xFFFFFFFF)],
                          ((seed & 0xFFFFFFFF) ^ (step >> 32), seed >> 32))
    for e in range(8):
        out[:, :, e] = (words[e // 2] >> np.uint64(16 * (e % 2))) & np.uint64(0xFFFF)
    return torch.from_numpy(out.reshape(rows, -1)[:, :width])


def threshold(p):
    return int(math.floor(65536 * p + 0.5))


def factor(rows, width, p, **kw):
    """0 where an element is dropped, else the scale (an fp32 value), float64."""
    t = threshold(p)
    scale = float(np.float32(65536 / (65536 - t))) if t < 65536 else 0.0
    return (draws(rows, width, **kw) >= t).double() * scale


def norm64(h, weight, bias, eps):
    mean = h.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((h - mean) ** 2).mean(-1, keepdim=True) + eps)
    hat = (h - mean) * rstd
    y = hat if weight is None else hat * weight
    return (y if bias is None else y + bias), mean, rstd, hat


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half the spacing of the type's subnormals: what a rounding of a tiny value may be off by."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def chain(width):
    """Longest chain of fp32 additions a row sum goes through, with the handful of roundings around it: at most 64
    elements of a row in one lane's running sum (the wide form has ceil(width / 2048) units of 8 more), then a tree."""
    return 64 + 16 + 8 * math.ceil(width / 2048)


def forward_bounds(h, weight, bias, eps, dtype):
    """(bound of y, bound of hat, relative bound of rstd) for rows h (float64, [rows, width]).

    mean: a chain of n additions of |h| <= m is off by at most n U mean|h| <= n U m; the subtraction and the scaling add 2 U
    of |hat|.  rstd: the variance is off by (n + 2) U of itself plus the square of the mean's error (part of the n U m
    term); its root halves that; 4 U for the root, the division and eps."""
    n = chain(h.shape[-1])
    y, mean, rstd, hat = norm64(h, weight, bias, eps)
    m = h.abs().mean(-1, keepdim=True)
    e_mean = n * U * m * rstd                       # the mean's error in units of hat
    e_rstd = (n / 2 + 6) * U + 0.5 * e_mean ** 2
    e_hat = e_mean + hat.abs() * (e_rstd + 3 * U)
    g = 1.0 if weight is None else weight.abs()
    b = 0.0 if bias is None else bias.abs()
    e_y = g * e_hat + 2 * U * (g * hat.abs() + b)
    return e_y + half_step(dtype) * (y.abs() + e_y) + tiny(dtype), e_hat, e_rstd


def backward_bounds(h, weight, dy, eps, e_hat, e_rstd):
    """(bound of rstd (t - mean t - hat mean(t hat)), bounds of the weight's and the bias's gradient) before the results'
    own rounding: every factor's error carried to first order, sums over a row as above, sums over rows through chains of
    at most 400 additions (128 rows of one partial sum and 256 partial sums, and the joins)."""
    n, r = chain(h.shape[-1]), 400
    _, _, rstd, hat = norm64(h, weight, None, eps)
    t = dy if weight is None else dy * weight
    mt, mth = t.abs().mean(-1, keepdim=True), (t * hat).abs().mean(-1, keepdim=True)
    c2 = (t * hat).mean(-1, keepdim=True).abs()
    e_c1 = (n + 2) * U * mt
    e_c2 = (n + 4) * U * mth + (t.abs() * e_hat).mean(-1, keepdim=True)
    inner = t.abs() + mt + hat.abs() * mth
    e_dx = rstd * (4 * U * inner + e_c1 + hat.abs() * e_c2 + c2 * e_hat) + rstd * inner * e_rstd
    e_dw = (dy.abs() * e_hat).sum(0) + (r + 3) * U * (dy * hat).abs().sum(0)
    e_db = r * U * dy.abs().sum(0)
    return e_dx, e_dw, e_db


def rounded(bound, value, dtype):
    return bound + half_step(dtype) * (value.abs() + bound) + tiny(dtype)


def close(got, want, bound, what):
    got, want, bound = got.detach().double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs() - bound * (1 + 1e-6)
    assert not torch.isnan(got).any(), what + " holds NaN"
    if off.numel():
        assert off.max() <= 0, "%s: off by %.3g more than its bound of %.3g at %d" % (
            what, off.max(), bound.flatten()[off.argmax()] if bound.numel() == off.numel() else bound.max(), off.argmax())
