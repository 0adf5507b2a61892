"""Binary64 forms of the norms between blocks and of the 8-bit products, with
bounds on what binary32 arithmetic can be off from them.

u = 2^-24 is half a step of binary32.  A sum of C terms is formed by up to 1024 threads
of at most 32 terms each, one after the other, then over the 64 lanes of a wave in
six levels, then over up to 16 waves one after the other: each term passes at most 32
+ 6 + 16 = 54 additions, so that a sum is off by at most 54 u times the sum of its
terms' magnitudes (to first order; squares are added unrounded).  SUM leaves ten
more, for the division and the second order.
"""
from __future__ import annotations

import numpy as np
from scipy import special

U = 2.0 ** -24
SUM = 64 * U
TYPES = {"f32": 0, "f16": 1, "bf16": 30, "i8": 24}
# half a step of a type, relative, and half its smallest step
HALF = {"f32": (2.0 ** -24, 2.0 ** -150), "f16": (2.0 ** -11, 2.0 ** -25),
        "bf16": (2.0 ** -8, 2.0 ** -134)}
NONE, RMS, LAYER = 0, 1, 2
ACTS = ("none", "silu", "gelu", "gelu_tanh", "relu", "sigmoid", "tanh")


def bf16_bits(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def store(x, kind):
    """(what the device holds, the values it stands for)"""
    x = np.asarray(x, np.float32)
    if kind == "f32":
        return np.ascontiguousarray(x), x.astype(np.float64)
    if kind == "f16":
        with np.errstate(over="ignore"):
            h = x.astype(np.float16)
        return h, h.astype(np.float64)
    u = bf16_bits(x)
    return u, (u.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def values(a, kind):
    if kind == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def act(kind, v):
    """(act(v), relative bound of binary32): exp and the like are a few steps off
    (erfc up to 16); their arguments' rounding counts as often as the function
    multiplies it: |z| for exp(z), 2 z^2 for erfc(z)."""
    v = np.asarray(v, np.float64)
    one = np.ones_like(v)
    if kind == "none":
        return v, 0 * one
    if kind == "relu":
        return np.maximum(v, 0.0), 0 * one
    with np.errstate(over="ignore", invalid="ignore"):
        if kind == "silu":
            return v * special.expit(v), 8 * U * one
        if kind == "sigmoid":
            return special.expit(v), 8 * U * one
        if kind == "tanh":
            return np.tanh(v), 8 * U * one
        if kind == "gelu":
            return 0.5 * v * special.erfc(-v / np.sqrt(2.0)), (40 + 4 * v * v) * U
        z = 2 * np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)
        return v * special.expit(z), (10 + 8 * np.abs(z)) * U


def norm(kind, eps, w, b, v, dv):
    """(the norm of rows v, its bound) where v itself may be dv off."""
    if kind == NONE:
        return v, dv
    C = v.shape[1]
    eps = float(np.float32(eps))
    if kind == LAYER:
        dmean = dv.mean(1, keepdims=True) + SUM * np.abs(v).mean(1, keepdims=True)
        v = v - v.mean(1, keepdims=True)
        dv = dv + dmean + U * np.abs(v)
    m = (v * v).mean(1, keepdims=True)
    dm = 2 * (np.abs(v) * dv).mean(1, keepdims=True) + (dv * dv).mean(1, keepdims=True) + SUM * m
    with np.errstate(divide="ignore", invalid="ignore"):
        r = 1 / np.sqrt(m + eps)
        rel = 0.75 * dm / (m + eps) + 6 * U        # half the sum's, and room for its square
    y = v * r
    dy = dv * r * (1 + rel) + np.abs(y) * rel
    if w is not None:
        y, dy = y * w, dy * np.abs(w) + np.abs(y * w) * U
    if b is not None:
        y, dy = y + b, dy + U * (np.abs(y) + np.abs(y + b))
    return y, dy


def block_norm(x, after, gate, gate_act, scale, residual, before):
    """sum, out and their binary32 bounds; after and before: (kind, eps, w, b)."""
    s, ds = norm(*after, x, np.zeros_like(x))
    if gate is not None:
        g, rel = act(gate_act, gate)
        ds = ds * np.abs(g) + np.abs(s * g) * (rel + U)
        s = s * g
    c = float(np.float32(scale))
    s, ds = s * c, ds * abs(c) + np.abs(s * c) * U
    if residual is not None:
        s = s + residual
        ds = ds + U * np.abs(s)
    out, dout = norm(*before, s, ds * 1.01)
    return s, ds * 1.01, out, dout * 1.01


def rounded(bound, want, kind):
    """A bound of binary32 results that are rounded to `kind` once."""
    rel, least = HALF[kind]
    return bound + (np.abs(want) + bound) * rel + least


def quantise(v):
    """Integers and scales of binary32 rows, exactly as promised: scale =
    max * binary32(1 / 127) in binary32, integers by the exact quotient, ties to even."""
    v = np.asarray(v, np.float32)
    most = np.abs(v).max(1)
    bad = ~np.isfinite(v).all(1)
    zero = ~bad & (most < np.float32(2.0 ** -100))
    scale = np.where(bad, np.float32(np.nan), np.where(zero, np.float32(0), most * (np.float32(1) / np.float32(127))))
    live = ~bad & ~zero
    q = np.zeros(v.shape, np.int8)
    # a quotient of two binary32 values is a half of an odd integer below 256 or
    # further than 2^-33 of itself from it: binary64's rounding keeps the side
    q[live] = np.rint(v[live].astype(np.float64) / scale[live, None].astype(np.float64)).astype(np.int8)
    return q, scale.astype(np.float32)


def product(q, xs, w, ws, bias=None):
    """The product as binary32 gives it, to the bit."""
    s = np.empty((q.shape[0], w.shape[0]), np.int64)
    # (sums below 2^53: binary64 products of integers are exact)
    s[:] = np.rint(q.astype(np.float64) @ w.astype(np.float64).T)
    with np.errstate(invalid="ignore", over="ignore"):
        y = s.astype(np.int32).astype(np.float32) * xs[:, None] * ws[None]
        if bias is not None:
            y = y + bias[None]
    return y.astype(np.float32)
