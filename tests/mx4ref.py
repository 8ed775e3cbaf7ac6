"""Plain 64-bit forms of the microscaled 4-bit rows, their products and the layer on them, and how far the kernels may be off.

Tolerances.  A block's products and their sum are exact; a matrix instruction adds two or four blocks to its 32-bit sum
and may be off by a step (2^-23) of the magnitudes so far, so a sum over nb blocks that at most eight others share is off by
less than (nb + 8) 2^-23 of the sum of magnitudes.  Everything after it is counted at its place."""
from __future__ import annotations

import numpy as np

from i8ref import EPS, round_rel

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])
STEP = 2.0 ** -23


def blocks(k):
    return (k + 31) // 32


def quantize(x):
    """x float32 [m][k] -> codes uint8 [m][32 * blocks] (one a byte) and scale bytes [m][blocks]."""
    x = np.asarray(x, np.float32).astype(np.float64)
    m, k = x.shape
    nb = blocks(k)
    x = np.pad(x, ((0, 0), (0, nb * 32 - k))).reshape(m, nb, 32)
    top = np.abs(x).max(2)
    fine = np.isfinite(x).all(2)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(fine & (top > 0), np.frexp(np.where(fine, top, 1.0))[1] - 1 - 2, -127)
    e = np.maximum(e, -127)
    v = np.where(fine[..., None], x, 0.0) * np.exp2(-e.astype(np.float64))[..., None]
    a = np.abs(v)[..., None]
    far = np.abs(a - VALUES[:8])
    best = far == far.min(-1, keepdims=True)           # one or two: the even code of two
    code = np.where(best.sum(-1) == 1, best.argmax(-1), np.where(best.argmax(-1) % 2 == 0, best.argmax(-1), best.argmax(-1) + 1))
    code = np.where(a[..., 0] >= 6, 7, code)
    code = code + 8 * np.signbit(v)
    code = np.where(fine[..., None], code, 0)
    return code.reshape(m, -1).astype(np.uint8), np.where(fine, e + 127, 255).astype(np.uint8)


def pack(codes):
    return (codes[..., 0::2] | codes[..., 1::2] << 4).astype(np.uint8)


def unpack(q):
    c = np.empty((*q.shape[:-1], 2 * q.shape[-1]), np.uint8)
    c[..., 0::2], c[..., 1::2] = q & 15, q >> 4
    return c


def values(q, s, k):
    """What packed rows and scale bytes stand for, float64 [..][k]."""
    v = VALUES[unpack(q)].reshape(*q.shape[:-1], -1, 32)
    scale = np.where(s == 255, np.nan, np.exp2(s.astype(np.float64) - 127))
    return (v * scale[..., None]).reshape(*q.shape[:-1], -1)[..., :k]


def sum_tol(x, w):
    """x [m][k] times w [r][k]: (nb + 8) steps of the magnitudes."""
    return (blocks(x.shape[1]) + 8) * STEP * (np.abs(x) @ np.abs(w).T)


def gemm_tol(y, tol, dtype, bias=None, old=None):
    a, err = np.abs(y), tol
    for more in (bias, old):
        if more is not None:
            a = a + np.abs(more)
            err = err + 1.01 * EPS["f32"] * a
    return err + 1.01 * round_rel(a, dtype)


def silu(g):
    return g / (1.0 + np.exp(-g))


def swiglu_tol(g, u, eg, eu, dtype):
    """|silu'| < 1.1; the exponential is within 2^-22 (|g| < 80), four more roundings follow it."""
    s = np.abs(silu(g))
    h = s * np.abs(u)
    return 1.1 * eg * np.abs(u) + s * eu + 1.1 * eg * eu + 8.1 * EPS["f32"] * h + 1.01 * round_rel(h, dtype)


def spread(x):
    """Each value's block's largest magnitude, [m][k]."""
    m, k = x.shape
    nb = blocks(k)
    top = np.abs(np.pad(x, ((0, 0), (0, nb * 32 - k))).reshape(m, nb, 32)).max(2)
    return top.repeat(32, 1)[:, :k]


def parts_tol(x, w):
    """x [m][k], split into nine parts, times w [r][k]: a value's parts have less than 1.3 of its block's largest magnitude M
    between them and leave 2^-26 M; nine columns are added."""
    return (1.3 * (blocks(x.shape[1]) + 17) * STEP + 2.0 ** -26) * (spread(x) @ np.abs(w).T)


def layer(x, gate, up, down, ids, w, dtype):
    """x [m][H]; gate / up / down float64 [n][..][..]; ids, w [m][slots] (id -1: none) -> y and its tolerance.  Weights are
    within 2^-21 (a sigmoid or softmax by a clamped exponential, or 64 bits rounded once)."""
    m, H = x.shape
    y, tol = np.zeros((m, H)), np.zeros((m, H))
    for t in range(m):
        mag = np.zeros(H)
        for e, share in zip(ids[t], w[t]):
            if e < 0:
                continue
            xt = x[t:t + 1]
            g, u = xt @ gate[e].T, xt @ up[e].T
            h = silu(g) * u
            eh = swiglu_tol(g, u, parts_tol(xt, gate[e]), parts_tol(xt, up[e]), "f32")
            v = (h @ down[e].T)[0]
            ev = (eh @ np.abs(down[e]).T + parts_tol(np.abs(h) + eh, down[e]))[0]
            y[t] += share * v
            mag += np.abs(share * v)
            tol[t] += np.abs(share) * ev + 2.0 ** -21 * np.abs(share * v)
        tol[t] += len(ids[t]) * EPS["f32"] * mag
    return y, tol + 1.01 * round_rel(np.abs(y) + tol, dtype)
