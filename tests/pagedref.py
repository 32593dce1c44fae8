"""Plain 64-bit forms of the rotary and paged-cache operators, for their tests."""
import numpy as np


def rotate(x, cos, sin, rot, neox, sign=1.0):
    """x [n, heads, hd] float64, cos/sin [n, rot/2] -> (y, bound on |fp32 result - y| before any rounding to 16 bits).

    Two products and one sum, each off by at most 2^-24 of its magnitude."""
    c, s = cos[:, None].astype(np.float64), sign * sin[:, None].astype(np.float64)
    y, err = x.copy(), np.zeros_like(x)
    h = rot // 2
    i0 = np.arange(h) if neox else 2 * np.arange(h)
    i1 = i0 + (h if neox else 1)
    x0, x1 = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    e0, e1 = np.abs(x0 * c) + np.abs(x1 * s), np.abs(x0 * s) + np.abs(x1 * c)
    err[..., i0], err[..., i1] = 2.01 * 2.0 ** -24 * e0, 2.01 * 2.0 ** -24 * e1
    return y, err


def rmsnorm(x, w, eps):
    """(x / sqrt(mean x^2 + eps) * w, relative bound): hd squares summed in fp32 (each partial sum off by
    2^-24, at most hd of them, halved by the square root), a square root, a quotient and two products."""
    hd = x.shape[-1]
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    return y, (hd / 2 + 5) * 2.0 ** -24


def attention(q, k, v, n_past, scale, u_p, tiny_p):
    """Causal attention of q [n, hd] over rows 0..n_past+i of k, v (float64) -> (out, bound on |fp32 result - out|).

    The kernel's error: each weight p = exp(s - max) <= 1 is rounded to 16 bits (relative u_p, at least tiny_p
    absolute); a score is a sum of hd products accumulated in fp32, off by at most hd 2^-23 sum|q k|, which
    multiplies its weight by exp of that (in numerator and sum); the exponential is off by 2^-21; the n weights and
    the n products with V are added up in fp32, at most n/8 additions after one another, 2^-23 each."""
    n, hd = q.shape
    s = (q @ k.T) * scale
    mag = (np.abs(q) @ np.abs(k).T) * scale
    hidden = np.arange(k.shape[0])[None] > (n_past + np.arange(n))[:, None]
    s = np.where(hidden, -np.inf, s)
    p = np.exp(s - s.max(-1, keepdims=True))
    l = p.sum(-1, keepdims=True)
    out = (p @ v) / l
    absv = np.abs(v)
    delta = np.where(hidden, 0.0, hd * 2.0 ** -23 * mag).max(-1, keepdims=True)
    rel = 2 * delta + 2 * 2.0 ** -21 + 2 * (k.shape[0] / 8 + 16) * 2.0 ** -23
    rounded = np.where(hidden, 0.0, np.maximum(u_p * p, tiny_p))
    return out, (rounded @ absv) / l + rel * ((p @ absv) / l)
