"""Plain 64-bit forms of routing by scores and of the int8 products with a scale per token and per channel."""
from __future__ import annotations

import numpy as np

EPS = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative
LEAST = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}  # a step of the smallest numbers


def torch_dtype(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def round_rel(y, dtype):
    """What rounding to `dtype` may move y by."""
    return EPS[dtype] * np.abs(y) + LEAST[dtype]


def route(logits, k, bias, score, n_group, topk_group, group_top, renorm, factor):
    """One row at a time, keys in float64, by sorting (key descending, index ascending)."""
    logits = np.asarray(logits, np.float64)
    m, E = logits.shape
    ids, w, n = np.full((m, k), -1, np.int64), np.zeros((m, k)), np.zeros(m, np.int64)
    for t in range(m):
        l = logits[t]
        free = l > -np.inf
        if score == "sigmoid":
            with np.errstate(over="ignore"):
                s = 1.0 / (1.0 + np.exp(-l))
        else:
            mx = l[free].max() if free.any() else 0.0
            e = np.where(free, np.exp(np.where(free, l, mx) - mx), 0.0)
            s = e / e.sum() if free.any() else e
        worth = s + (0.0 if bias is None else np.asarray(bias, np.float64))
        key = l if bias is None else worth
        free = free & (key > -np.inf)
        gs = E // n_group
        if n_group > 1:
            gw = []
            for g in range(n_group):
                of = (worth if group_top == 2 else key)[g * gs:(g + 1) * gs][free[g * gs:(g + 1) * gs]]
                gw.append(np.sort(of)[::-1][:group_top].sum() if of.size else -np.inf)
            order = sorted((g for g in range(n_group) if gw[g] > -np.inf), key=lambda g: (-gw[g], g))[:topk_group]
            free = free & np.isin(np.arange(E) // gs, order)
        best = sorted(np.nonzero(free)[0], key=lambda e: (-key[e], e))[:k]
        n[t] = len(best)
        ids[t, :n[t]] = best
        ws = s[best]
        if renorm:
            ws = ws / ws.sum() if ws.size and ws.sum() > 0 else ws * 0
        w[t, :n[t]] = ws * factor
    return ids, w, n


def quantize(x):
    """x (any float array [m][k], finite) -> q, scale; the quotients in 64-bit mantissas."""
    x = np.asarray(x, np.float64)
    top = np.abs(x).max(1)
    live = top >= 127 * 2.0 ** -126
    safe = np.where(live, top, 1.0)
    q = np.rint(np.longdouble(127) * x.astype(np.longdouble) / safe.astype(np.longdouble)[:, None])
    return np.where(live[:, None], q, 0).astype(np.int8), np.where(live, safe / 127, 0).astype(np.float32)


def gemm(q, s, w, ws):
    """Exact integer sums, scaled in float64."""
    acc = q.astype(np.float64) @ w.astype(np.float64).T  # exact: below 2^53
    return acc * np.asarray(s, np.float64)[:, None] * np.asarray(ws, np.float64)


def gemm_tol(y, dtype, bias=None, old=None):
    """trk_gemm_i8: three roundings of the product (sum to 32 bits, times s_x, times s_w), one for each sum, then the output's."""
    a = np.abs(y)
    err = 3.01 * EPS["f32"] * a
    for more in (bias, old):
        if more is not None:
            a = a + np.abs(more)
            err = err + 1.01 * EPS["f32"] * a
    return err + 1.01 * round_rel(a, dtype)


def swiglu(g, u):
    return g / (1.0 + np.exp(-g)) * u


def swiglu_tol(g, u, dtype):
    """g and u within 3 half steps each; silu multiplies g's relative error by 1 + |g| at most; the exponential is within
    2^-22 (its clamped polynomial, |g| < 80), and four more roundings follow it."""
    h = np.abs(swiglu(g, u))
    return h * ((3 * (1 + np.abs(g)) + 3 + 4 + 4) * 1.01 * EPS["f32"]) + 1.01 * round_rel(h, dtype)


def entries(ids, n, slots, E):
    """[m][slots] truth values: which slots are entries."""
    ids, n = np.asarray(ids)[:, :slots], np.asarray(n)
    return (np.arange(slots)[None, :] < n[:, None]) & (ids >= 0) & (ids < E)
