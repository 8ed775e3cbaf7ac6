"""Microscaled 4-bit rows, their products and the layer on them, on the GPU, against plain 64-bit forms (tests/mx4ref.py)."""
from __future__ import annotations

import sys

import i8ref
import mx4ref as R
import numpy as np
import pytest

import trmoe

pytestmark = pytest.mark.gpu
DTYPES = ["f32", "bf16", "f16"]


def say(msg):
    print(f"[gpu] {msg}", flush=True)
    sys.stdout.flush()


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    return t.detach().float().cpu().numpy() if t.is_floating_point() else t.detach().cpu().numpy()


def rows4(rng, *shape, spread=1.0):
    """Packed rows and scales [..][k] of values near `spread`, their blocks a few powers of two apart, as host arrays."""
    *lead, k = shape
    m, nb = int(np.prod(lead)), R.blocks(k)
    v = rng.standard_normal((m, nb * 32), dtype=np.float32) * 2
    codes = np.searchsorted(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32), np.abs(v)).astype(np.uint8)
    codes += np.where(v < 0, 8, 0).astype(np.uint8)
    codes[:, k:] = 0
    s = 126 + int(np.rint(np.log2(spread))) + rng.integers(-3, 4, (m, nb))
    return R.pack(codes).reshape(*lead, -1), s.astype(np.uint8).reshape(*lead, -1)


def apart(q, s, more=1):
    """The same on the GPU with 16 * more bytes behind each row of values and 4 * more behind its scales (up to a multiple of
    4 at least), all ones: a scale byte of NaN."""
    import torch
    nb = s.shape[-1]
    qt = torch.full((*q.shape[:-1], q.shape[-1] + 16 * more), 255, dtype=torch.uint8, device="cuda")
    st = torch.full((*s.shape[:-1], (nb + 3) // 4 * 4 + 4 * more), 255, dtype=torch.uint8, device="cuda")
    qt[..., :q.shape[-1]], st[..., :nb] = dev(q), dev(s)
    return qt[..., :q.shape[-1]], st[..., :nb]


def within(got, want, tol):
    assert np.isfinite(got).all()
    bad = np.abs(got - want) > tol
    assert not bad.any(), f"{bad.sum()} of {bad.size}: worst {np.max(np.abs(got - want) / tol):.3g} of the bound at {np.argwhere(bad)[0]}"


# ---- rows to 4-bit values, and back ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,lead,spare", [(1, 1, 0, 0), (3, 31, 0, 1), (5, 32, 1, 0), (2, 33, 0, 0), (70, 96, 3, 5), (4, 2048, 0, 0),
                                            (9, 1000, 0, 24), (300, 100, 0, 0), (2, 8191, 1, 0), (1, 70000, 0, 0)])
def test_quantize_and_back(dtype, m, k, lead, spare):
    import torch
    say(f"quantize_mx4 {dtype} {m} x {k}")
    rng = np.random.default_rng(k + m)
    wide = rng.standard_normal((m, lead + k + spare)) * np.exp2(rng.integers(-12, 8, (m, 1)))
    wide[:, ::7] = np.round(wide[:, ::7] * 4) / 4  # on the borders, many of them
    if m > 2:
        wide[1] = 0
    t = dev(wide.astype(np.float32)).to(i8ref.torch_dtype(dtype))[:, lead:lead + k]
    nb = R.blocks(k)
    q = torch.full((m, 16 * nb + 32), 77, dtype=torch.uint8, device="cuda")
    s = torch.full((m, (nb + 3) // 4 * 4 + 4), 77, dtype=torch.uint8, device="cuda")
    trmoe.quantize_mx4(t, out=(q[:, :16 * nb], s[:, :nb]))
    codes, scale = R.quantize(host(t))
    assert np.array_equal(host(s)[:, :nb], scale) and np.array_equal(host(q)[:, :16 * nb], R.pack(codes))
    assert (host(q)[:, 16 * nb:] == 77).all() and (host(s)[:, nb:] == 77).all()
    q2, s2 = trmoe.quantize_mx4(t)
    assert torch.equal(q2, q[:, :16 * nb]) and torch.equal(s2, s[:, :nb])
    for to in DTYPES:
        y = torch.full((m, k + 3), 5.0, dtype=i8ref.torch_dtype(to), device="cuda")
        trmoe.dequantize_mx4(q2, s2, k, out=y[:, 1:1 + k])
        want = dev(R.values(host(q2), scale, k).astype(np.float32)).to(y.dtype)
        assert torch.equal(y[:, 1:1 + k], want) and (y[:, 0] == 5).all() and (y[:, 1 + k:] == 5).all()
        assert torch.equal(trmoe.dequantize_mx4(q2, s2, k, dtype=y.dtype), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_poison_and_extremes(dtype):
    say(f"quantize_mx4 poison {dtype}")
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, 96)).astype(np.float32)
    x[0, 5], x[1, 40], x[2, 95] = np.nan, np.inf, -np.inf
    big, small = {"f32": (3.3e38, 1e-45), "bf16": (3.3e38, 1e-40), "f16": (65504.0, 6e-8)}[dtype]
    x[3, :32], x[4, 32:64] = x[3, :32] * 0 + big, x[4, 32:64] * small
    x[5] = np.tile([2.0 ** -125, 2.0 ** -126, -2.0 ** -127, 2.0 ** -128], 24)
    t = dev(x).to(i8ref.torch_dtype(dtype))
    q, s = trmoe.quantize_mx4(t)
    codes, scale = R.quantize(host(t))
    assert np.array_equal(host(s), scale) and np.array_equal(host(q), R.pack(codes))
    assert [host(s)[0, 0], host(s)[1, 1], host(s)[2, 2]] == [255] * 3
    y = host(trmoe.dequantize_mx4(q, s, 96))
    assert np.isnan(y[0, :32]).all() and np.isfinite(y[0, 32:]).all()


def test_dequantize_every_code_and_scale():
    import torch
    say("dequantize_mx4 every code and scale")
    q = np.tile(R.pack(np.tile(np.arange(16, dtype=np.uint8), 2)), (256, 1))
    s = np.arange(256, dtype=np.uint8)[:, None]
    qt, st = apart(q, s)
    with np.errstate(over="ignore"):
        want = R.values(q, s, 32).astype(np.float32)
    for to in DTYPES:
        got = trmoe.dequantize_mx4(qt, st, 32, dtype=i8ref.torch_dtype(to))
        assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(dev(want).to(got.dtype), nan=7.0))
        assert got[255].isnan().all()


# ---- the dense product -------------------------------------------------------------------------------

GEMMS = [(1, 1, 1), (1, 16, 32), (2, 17, 33), (3, 100, 128), (16, 31, 129), (17, 64, 500), (1, 5003, 1999), (33, 129, 257),
         (64, 64, 1024), (65, 300, 100), (100, 1000, 800), (130, 700, 1056), (300, 515, 2100), (513, 770, 300), (700, 2050, 544)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,rows,k", GEMMS)
def test_gemm(m, rows, k, dtype):
    say(f"gemm_mx4 {m} x {rows} x {k} {dtype}")
    rng = np.random.default_rng(m + rows + k)
    (q, s), (wq, ws) = rows4(rng, m, k), rows4(rng, rows, k)
    x, w = R.values(q, s, k), R.values(wq, ws, k)
    bias = rng.standard_normal(rows).astype(np.float32) if rows % 2 else None
    W = trmoe.MX4Weights(*apart(wq, ws), k)
    y = trmoe.gemm_mx4(W, *apart(q, s, 2), bias=None if bias is None else dev(bias), dtype=i8ref.torch_dtype(dtype))
    want = x @ w.T
    tol = R.gemm_tol(want, R.sum_tol(x, w), dtype, bias)
    within(host(y), want if bias is None else want + bias, tol)


@pytest.mark.parametrize("m,rows,k,bias,acc", [(4000, 4000, 2100, False, False), (4096, 4096, 2080, True, False), (4001, 4003, 300, True, True)])
def test_gemm_large(m, rows, k, bias, acc):
    """Tiles of 256 x 256, whole and ragged: several groups of scales, a bias, an output that is added to."""
    import torch
    say(f"gemm_mx4 large {m} x {rows} x {k}")
    rng = np.random.default_rng(3)
    (q, s), (wq, ws) = rows4(rng, m, k), rows4(rng, rows, k)
    W, xs = trmoe.MX4Weights(*apart(wq, ws), k), apart(q, s)
    b = rng.standard_normal(rows).astype(np.float32) if bias else None
    old = torch.randn((m, rows), device="cuda") if acc else None
    y = trmoe.gemm_mx4(W, *xs, bias=None if b is None else dev(b), out=None if old is None else old.clone(), accumulate=acc)
    x, w = dev(R.values(q, s, k)), dev(R.values(wq, ws, k))  # in 64 bits on the GPU
    want, mag = x @ w.T, x.abs() @ w.abs().T
    tol = (R.blocks(k) + 8) * R.STEP * mag + 2 ** -23 * want.abs()
    if bias:
        want, tol = want + dev(b).double(), tol + 2 ** -23 * (want.abs() + dev(b).abs())
    if acc:
        want, tol = want + old.double(), tol + 2 ** -23 * (want.abs() + old.abs())
    far = ((y.double() - want).abs() / (tol + 1e-30)).max().item()
    assert far <= 1, far


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,rows,k", [(3, 50, 70), (200, 300, 160)])
def test_gemm_accumulates_and_takes_an_item(dtype, m, rows, k):
    import torch
    say(f"gemm_mx4 accumulate {m} x {rows} x {k} {dtype}")
    rng = np.random.default_rng(7)
    (q, s), (wq, ws) = rows4(rng, m, k), rows4(rng, 3, rows, k)
    x, w = R.values(q, s, k), R.values(wq[2], ws[2], k)
    W = trmoe.MX4Weights(*apart(wq, ws), k)
    wide = torch.randn((m, rows + 5), device="cuda").to(i8ref.torch_dtype(dtype))
    old, before = host(wide[:, 1:1 + rows]), wide.clone()
    trmoe.gemm_mx4(W, *apart(q, s), out=wide[:, 1:1 + rows], accumulate=True, item=2)
    want = x @ w.T
    within(host(wide[:, 1:1 + rows]), want + old, R.gemm_tol(want, R.sum_tol(x, w), dtype, old=old))
    assert torch.equal(wide[:, 0], before[:, 0]) and torch.equal(wide[:, 1 + rows:], before[:, 1 + rows:])


@pytest.mark.parametrize("m,rows", [(3, 20), (300, 300)])
def test_gemm_poison_stays_in_its_row(m, rows):
    say(f"gemm_mx4 poison {m} x {rows}")
    rng = np.random.default_rng(1)
    k = 300
    (q, s), (wq, ws) = rows4(rng, m, k), rows4(rng, rows, k)
    s[1, 9], ws[7, 0] = 255, 255
    y = host(trmoe.gemm_mx4(trmoe.MX4Weights(*apart(wq, ws), k), *apart(q, s)))
    nan = np.zeros((m, rows), bool)
    nan[1], nan[:, 7] = True, True
    assert np.array_equal(np.isnan(y), nan)


def test_gemm_scales_of_any_size():
    """Scales whose product alone leaves 32 bits' range in either direction."""
    say("gemm_mx4 far scales")
    rng = np.random.default_rng(5)
    (q, s), (wq, ws) = rows4(rng, 20, 256), rows4(rng, 40, 256)
    for a, b in ((0, 254), (254, 0), (1, 200), (60, 100), (127 + 60, 127 - 60)):
        s[:], ws[:] = a, b
        x, w = R.values(q, s, 256), R.values(wq, ws, 256)
        y = host(trmoe.gemm_mx4(trmoe.MX4Weights(dev(wq), dev(ws), 256), dev(q), dev(s)))
        within(y, x @ w.T, R.gemm_tol(x @ w.T, R.sum_tol(x, w), "f32"))


def test_gemm_one_row_of_any_stride():
    """A single row, and a matrix of one, have no stride to obey."""
    import torch
    say("gemm_mx4 single rows")
    rng = np.random.default_rng(6)
    (q, s), (wq, ws) = rows4(rng, 4, 160), rows4(rng, 1, 160)
    qt, st = dev(q), torch.zeros((4, 7), dtype=torch.uint8, device="cuda")  # rows of scales 7 bytes apart
    st.view(-1)[0:5] = dev(s[0])
    x, w = R.values(q[:1], s[:1], 160), R.values(wq, ws, 160)
    W = trmoe.MX4Weights(dev(wq), torch.cat((dev(ws), dev(ws)), 1)[:, :5], 160)
    y = trmoe.gemm_mx4(W, qt[:1], st[:1, :5])
    within(host(y), x @ w.T, R.gemm_tol(x @ w.T, R.sum_tol(x, w), "f32"))
    with pytest.raises(trmoe.TrkError, match="4-byte pieces|multiples of 4"):
        trmoe.gemm_mx4(W, qt, st[:, :5])


# ---- the experts' products ---------------------------------------------------------------------------

def routing(rng, m, E, slots, kind):
    """ids / w [m][32] and n_sel [m]; kind: even, one (everybody's first expert alike), ragged (n from 0), foreign (ids past
    the stack)."""
    ids = np.full((m, 32), 0x7fffffff, np.int32)
    w = np.zeros((m, 32), np.float32)
    for t in range(m):
        ids[t, :slots] = rng.permutation(max(E, slots))[:slots] % E
    w[:, :slots] = rng.uniform(0.05, 1.0, (m, slots))
    n = np.full(m, slots, np.int32)
    if kind == "one":
        ids[:, 0] = E - 1
    if kind == "ragged":
        n = rng.integers(0, slots + 1, m).astype(np.int32)
        n[0] = 0
    if kind == "foreign":
        ids[rng.random((m, 32)) < 0.3] = E + 3
        ids[rng.random((m, 32)) < 0.1] = -1
    return ids, w, n


EXPERTS = [(1, 4, 2, 64, 48, "even"), (3, 8, 8, 100, 33, "ragged"), (8, 16, 10, 300, 70, "foreign"), (9, 8, 2, 96, 64, "even"),
           (40, 5, 3, 130, 100, "one"), (64, 64, 4, 544, 129, "ragged"), (100, 16, 4, 256, 200, "foreign"),
           (200, 4, 2, 320, 272, "one"), (300, 7, 3, 1100, 90, "even"), (700, 3, 2, 200, 300, "ragged"), (30, 300, 6, 64, 40, "even"),
           (9, 1, 1, 33, 17, "even"), (1500, 12, 4, 96, 96, "one")]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,E,slots,H,F,kind", EXPERTS)
def test_experts_up(m, E, slots, H, F, kind, dtype):
    import torch
    say(f"experts_up_mx4 m={m} E={E} slots={slots} H={H} F={F} {kind} {dtype}")
    rng = np.random.default_rng(m + E + H)
    (q, s), (gq, gs), (uq, us) = rows4(rng, m, H), rows4(rng, E, F, H, spread=H ** -0.5), rows4(rng, E, F, H, spread=H ** -0.5)
    ids, w, n = routing(rng, m, E, slots, kind)
    x, gate, up = R.values(q, s, H), R.values(gq, gs, H), R.values(uq, us, H)
    idt, nt = dev(ids), dev(n)
    out = torch.full((m * slots, F + 2), 9.0, dtype=i8ref.torch_dtype(dtype), device="cuda")
    plan = trmoe.experts_plan(idt, nt, slots, E)
    trmoe.experts_up_mx4(trmoe.MX4Weights(*apart(gq, gs), H), trmoe.MX4Weights(*apart(uq, us, 2), H), *apart(q, s), idt, nt, slots,
                         plan=plan, out=out[:, 1:1 + F])
    got, there = host(out), i8ref.entries(ids, n, slots, E)
    assert (got[:, 0] == 9).all() and (got[:, 1 + F:] == 9).all() and (got[~there.reshape(-1)] == 9).all()
    for e in range(E):
        t, j = np.nonzero(there & (ids[:, :slots] == e))
        if not t.size:
            continue
        g, u = x[t] @ gate[e].T, x[t] @ up[e].T
        tol = R.swiglu_tol(g, u, R.sum_tol(x[t], gate[e]), R.sum_tol(x[t], up[e]), dtype)
        within(got[t * slots + j][:, 1:1 + F], R.silu(g) * u, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,E,slots,F,H,kind", EXPERTS)
def test_experts_down(m, E, slots, F, H, kind, dtype):
    import torch
    say(f"experts_down_mx4 m={m} E={E} slots={slots} F={F} H={H} {kind} {dtype}")
    rng = np.random.default_rng(m + E + F)
    (q, s), (wq, ws) = rows4(rng, m * slots, F), rows4(rng, E, H, F)
    ids, w, n = routing(rng, m, E, slots, kind)
    x, down = R.values(q, s, F), R.values(wq, ws, F)
    idt, nt, wt = dev(ids), dev(n), dev(w)
    W, qs = trmoe.MX4Weights(*apart(wq, ws), F), apart(q, s)
    plan = trmoe.experts_plan(idt, nt, slots, E)
    y = trmoe.experts_down_mx4(W, *qs, idt, wt, nt, slots, plan=plan, dtype=i8ref.torch_dtype(dtype))
    want, tol, mag = np.zeros((m, H)), np.zeros((m, H)), np.zeros((m, H))
    there = i8ref.entries(ids, n, slots, E)
    for e in range(E):
        t, j = np.nonzero(there & (ids[:, :slots] == e))
        if not t.size:
            continue
        share = w[t, j].astype(np.float64)[:, None]
        v = x[t * slots + j] @ down[e].T * share
        np.add.at(want, t, v), np.add.at(mag, t, np.abs(v))
        np.add.at(tol, t, R.sum_tol(x[t * slots + j], down[e]) * share)
    tol = tol + (slots + 2) * i8ref.EPS["f32"] * mag
    within(host(y), want, tol + 1.01 * i8ref.round_rel(mag + tol, dtype))
    before = y.clone()
    trmoe.experts_down_mx4(W, *qs, idt, wt, nt, slots, plan=plan, out=y, accumulate=True)
    old = host(before).astype(np.float64)
    within(host(y), want + old, tol + 1.01 * i8ref.EPS["f32"] * (mag + np.abs(old)) + 1.01 * i8ref.round_rel(mag + tol + np.abs(old), dtype))
    assert (want[n == 0] == 0).all() and (host(before)[n == 0] == 0).all()


# m, E, slots, k, rows (of gate and up, or of down): every shape of tile, several stages and groups of scales
MANY = [(300, 200, 4, 1100, 272, "even"), (500, 64, 4, 640, 400, "ragged"), (1000, 64, 4, 2100, 390, "even"),
        (2000, 16, 4, 416, 512, "one"), (60, 20, 2, 2100, 96, "foreign"), (120, 12, 4, 1300, 130, "even"), (900, 8, 2, 1600, 80, "even")]


@pytest.mark.parametrize("m,E,slots,k,rows,kind", MANY)
def test_experts_of_many_entries(m, E, slots, k, rows, kind):
    import torch
    say(f"experts mx4 many m={m} E={E} slots={slots} k={k} rows={rows} {kind}")
    rng = np.random.default_rng(m + E)
    (gq, gs), (uq, us) = rows4(rng, E, rows, k, spread=k ** -0.5), rows4(rng, E, rows, k, spread=k ** -0.5)
    (xq, xs), (hq, hs) = rows4(rng, m, k), rows4(rng, m * slots, k)
    ids, w, n = routing(rng, m, E, slots, kind)
    idt, nt, wt = dev(ids), dev(n), dev(w)
    plan = trmoe.experts_plan(idt, nt, slots, E)
    G, U = trmoe.MX4Weights(*apart(gq, gs), k), trmoe.MX4Weights(*apart(uq, us), k)
    h = torch.full((m * slots, rows), 9.0, device="cuda")
    trmoe.experts_up_mx4(G, U, *apart(xq, xs), idt, nt, slots, plan=plan, out=h)
    y = host(trmoe.experts_down_mx4(G, *apart(hq, hs), idt, wt, nt, slots, plan=plan))
    x, x2, gate, up = R.values(xq, xs, k), R.values(hq, hs, k), R.values(gq, gs, k), R.values(uq, us, k)
    there, got = i8ref.entries(ids, n, slots, E), host(h)
    assert (got[~there.reshape(-1)] == 9).all()
    want, tol, mag = np.zeros((m, rows)), np.zeros((m, rows)), np.zeros((m, rows))
    for e in range(E):
        t, j = np.nonzero(there & (ids[:, :slots] == e))
        if not t.size:
            continue
        g, u = x[t] @ gate[e].T, x[t] @ up[e].T
        within(got[t * slots + j], R.silu(g) * u, R.swiglu_tol(g, u, R.sum_tol(x[t], gate[e]), R.sum_tol(x[t], up[e]), "f32"))
        share, rows_ = w[t, j].astype(np.float64)[:, None], x2[t * slots + j]
        v = rows_ @ gate[e].T * share
        np.add.at(want, t, v), np.add.at(mag, t, np.abs(v)), np.add.at(tol, t, R.sum_tol(rows_, gate[e]) * share)
    tol = tol + (slots + 2) * i8ref.EPS["f32"] * mag
    within(y, want, tol + 1.01 * i8ref.round_rel(mag + tol, "f32"))


@pytest.mark.parametrize("call", ["up", "down"])
@pytest.mark.parametrize("made", [(100, 2, 8), (90, 3, 8), (100, 3, 9)])
def test_a_plan_of_another_call(call, made):
    """A plan made for another m, slots or number of experts, of as many words or more, is not followed: what it would write is
    NaN, and nothing else is written."""
    import torch
    say(f"experts mx4 {call} with a plan of {made}")
    rng = np.random.default_rng(5)
    m, slots, E, k, rows = 100, 3, 8, 96, 64
    ids, w, n = routing(rng, m, E, slots, "ragged")
    idt, nt, wt = dev(ids), dev(n), dev(w)
    oids, _, on = routing(rng, made[0], made[2], made[1], "even")
    words = trmoe._plan_words(m, slots, E)
    plan = torch.zeros(words + 4096, dtype=torch.int32, device="cuda")
    other = trmoe.experts_plan(dev(oids), dev(on), made[1], made[2])
    plan[:other.numel()] = other[:plan.numel()]
    plan = plan[:words].contiguous()
    G = trmoe.MX4Weights(*apart(*rows4(rng, E, rows, k)), k)
    there = i8ref.entries(ids, n, slots, E)
    if call == "up":
        h = torch.full((m * slots, rows), 9.0, device="cuda")
        trmoe.experts_up_mx4(G, G, *apart(*rows4(rng, m, k)), idt, nt, slots, plan=plan, out=h)
        got = host(h)
        assert np.isnan(got[there.reshape(-1)]).all() and (got[~there.reshape(-1)] == 9).all()
    else:
        y = host(trmoe.experts_down_mx4(G, *apart(*rows4(rng, m * slots, k)), idt, wt, nt, slots, plan=plan))
        assert np.isnan(y[there.any(1)]).all() and (y[~there.any(1)] == 0).all()


def test_rows_far_apart():
    """Rows whose tiles' 32-bit offsets would not hold them go entry by entry, tile by strip."""
    import torch
    say("mx4 rows far apart")
    rng = np.random.default_rng(6)
    m, E, slots, k, rows = 40, 3, 2, 96, 40
    (wq, ws), (xq, xs) = rows4(rng, E, rows, k), rows4(rng, m, k)
    ids, w, n = routing(rng, m, E, slots, "even")
    plan = trmoe.experts_plan(dev(ids), dev(n), slots, E)
    near = trmoe.MX4Weights(dev(wq), apart(wq, ws, 0)[1], k)
    far = torch.zeros((E, rows, 1 << 23), dtype=torch.uint8, device="cuda")[:, :, :48]
    far.copy_(dev(wq))
    F = trmoe.MX4Weights(far, near.scale, k)
    sx = torch.zeros((m, 1 << 23), dtype=torch.uint8, device="cuda")[:, :3]
    sx.copy_(dev(xs))
    x, xn = (dev(xq), sx), (dev(xq), apart(xq, xs, 0)[1])
    for W, rowsx in ((F, xn), (near, x), (F, x)):
        assert torch.equal(trmoe.gemm_mx4(W, *rowsx, item=1), trmoe.gemm_mx4(near, *xn, item=1))
        a = trmoe.experts_up_mx4(W, near, *rowsx, dev(ids), dev(n), slots, plan=plan)
        b = trmoe.experts_up_mx4(near, near, *xn, dev(ids), dev(n), slots, plan=plan)
        tol = 1e-5 * b.abs().max()
        assert (a - b).abs().max() <= tol


# ---- the layer ---------------------------------------------------------------------------------------

def layer_of(rng, E, H, F, n_shared=0, gated=False, bias=False, router=True):
    n = E + n_shared
    w = {"gate": rows4(rng, n, F, H, spread=0.3 * H ** -0.5), "up": rows4(rng, n, F, H, spread=0.3 * H ** -0.5),
         "down": rows4(rng, n, H, F, spread=0.3 * F ** -0.5)}
    r = (rng.standard_normal((E, H)) * 1.3 / H ** 0.5).astype(np.float32) if router else None
    b = (rng.standard_normal(E) * 0.05).astype(np.float32) if bias else None
    sg = (rng.standard_normal(H) / H ** 0.5).astype(np.float32) if gated else None
    k = {"gate": H, "up": H, "down": F}
    L = trmoe.MX4Layer(*[trmoe.MX4Weights(*apart(*w[i]), k[i]) for i in ("gate", "up", "down")],
                       router=None if r is None else dev(r), bias=None if b is None else dev(b), n_shared=n_shared,
                       shared_gate=None if sg is None else dev(sg))
    return L, {i: R.values(*w[i], k[i]) for i in w}, r, b, sg


@pytest.mark.parametrize("m,E,k,H,F,shared,gated,bias,score,groups,keep,xt,yt", [
    (1, 4, 2, 64, 32, 0, False, False, "softmax", 1, 1, "f32", "f32"), (1, 24, 10, 2048, 512, 1, True, False, "softmax", 1, 1, "bf16", "f32"),
    (8, 64, 8, 300, 96, 2, False, True, "sigmoid", 8, 4, "f32", "f32"), (3, 10, 2, 650, 215, 0, False, False, "softmax", 1, 1, "f16", "f16"),
    (5, 7, 7, 33, 700, 1, True, True, "sigmoid", 1, 1, "bf16", "bf16"), (2, 33, 32, 130, 65, 32, False, False, "softmax", 1, 1, "f32", "f16"),
    (8, 8, 8, 4100, 40, 0, False, True, "softmax", 2, 1, "f32", "bf16"), (4, 1, 1, 1, 1, 0, False, False, "sigmoid", 1, 1, "f32", "f32"),
    (7, 1024, 4, 96, 128, 3, True, False, "sigmoid", 4, 2, "f16", "f32"), (6, 16, 5, 2049, 1056, 0, False, False, "sigmoid", 1, 1, "bf16", "f32")])
def test_layer(m, E, k, H, F, shared, gated, bias, score, groups, keep, xt, yt):
    import torch
    if E // groups * keep < k:
        k = E // groups * keep
    say(f"moe_mx4 m={m} E={E} k={k} H={H} F={F} shared={shared} {score} {xt} {yt}")
    rng = np.random.default_rng(m * 100 + E + H)
    L, w, r, b, sg = layer_of(rng, E, H, F, shared, gated, bias)
    wide = dev((rng.standard_normal((m, H + 7)) * np.exp2(rng.integers(-2, 3, (m, 1)))).astype(np.float32)).to(i8ref.torch_dtype(xt))
    xd = wide[:, 3:3 + H]
    x = host(xd).astype(np.float64)
    kw = dict(k=k, n_group=groups, topk_group=keep, group_top=2, renorm=True, factor=1.5)
    logits = x @ r.astype(np.float64).T
    rid, rw, rn = i8ref.route(logits, bias=b, score=score, **kw)
    for sign in (1, -1):  # the choice does not hang on the logits' last bits
        moved = logits + sign * 1e-6 * np.sign(rng.standard_normal(logits.shape)) * np.abs(logits).max()
        assert np.array_equal(i8ref.route(moved, bias=b, score=score, **kw)[0], rid)
    gatew = 1 / (1 + np.exp(-(x @ sg.astype(np.float64)))) if gated else np.ones(m)
    ids = np.concatenate((rid, np.tile(np.arange(E, E + shared), (m, 1))), 1)
    share = np.concatenate((rw, np.tile(gatew[:, None], (1, shared))), 1)
    want, tol = R.layer(x, w["gate"], w["up"], w["down"], ids, share, yt)
    # the logits: k products in 32 bits, and what moves with them, the weights and the shared gate
    eps = (H / 64 + 16) * R.STEP * (np.abs(x) @ np.abs(r).T).max() + (R.STEP * (H / 64 + 16) * (np.abs(x) @ np.abs(sg)).max() if gated else 0)
    tol = tol + 2 * eps * np.array([sum(abs(share[t, j]) * np.abs(R.silu(x[t] @ w["gate"][e].T) * (x[t] @ w["up"][e].T)) @ np.abs(w["down"][e]).T
                                        for j, e in enumerate(ids[t]) if e >= 0) for t in range(m)])
    y = torch.full((m, H + 2), 3.0, dtype=i8ref.torch_dtype(yt), device="cuda")
    trmoe.moe_mx4(L, xd, score=score, out=y[:, 1:1 + H], **kw)
    within(host(y)[:, 1:1 + H], want, tol)
    assert (y[:, 0] == 3).all() and (y[:, 1 + H:] == 3).all()
    # the logits given: the same experts
    y2 = trmoe.moe_mx4(L, xd, rlog=dev(logits.astype(np.float32)), score=score, dtype=torch.float32, **kw)
    within(host(y2), want, R.layer(x, w["gate"], w["up"], w["down"], ids, share, "f32")[1] + tol)


@pytest.mark.parametrize("m,E,k,H,F,shared", [(8, 40, 8, 512, 600, 1), (8, 16, 2, 1030, 1100, 0), (5, 300, 12, 640, 200, 2),
                                                (8, 30, 6, 1041, 70, 1), (7, 9, 5, 1200, 1100, 0), (8, 36, 32, 1039, 33, 21)])
def test_layer_of_many_entries(m, E, k, H, F, shared):
    """The choice by a launch of its own, several units of K, slots in turn."""
    say(f"moe_mx4 many m={m} E={E} k={k} H={H} F={F} shared={shared}")
    rng = np.random.default_rng(m + E + k)
    L, w, _, _, _ = layer_of(rng, E, H, F, shared, router=False)
    x = rng.standard_normal((m, H)).astype(np.float32) * np.exp2(rng.integers(-20, 20, (m, H // 2 + 1)).repeat(2, 1)[:, :H]).astype(np.float32)
    x = x / np.abs(x).max() * 4  # values far below their block's largest
    logits = (rng.permutation(m * E).reshape(m, E) / (m * E)).astype(np.float32)
    kw = dict(k=k, n_group=1, topk_group=1, group_top=2, renorm=False, factor=1.0)
    rid, rw, rn = i8ref.route(logits, bias=None, score="sigmoid", **kw)
    ids = np.concatenate((rid, np.tile(np.arange(E, E + shared), (m, 1))), 1)
    share = np.concatenate((rw, np.ones((m, shared))), 1)
    y = host(trmoe.moe_mx4(L, dev(x), rlog=dev(logits), score="sigmoid", **kw))
    want, tol = R.layer(x.astype(np.float64), w["gate"], w["up"], w["down"], ids, share, "f32")
    within(y, want, tol)


def test_layer_rows_that_choose_nothing():
    """A token whose logits leave no expert has its shared ones alone, or zeros; a poisoned token poisons itself."""
    import torch
    say("moe_mx4 masked rows")
    rng = np.random.default_rng(2)
    E, H, F, m = 6, 96, 64, 5
    for shared in (0, 1):
        L, w, _, _, _ = layer_of(rng, E, H, F, shared, router=False)
        x = rng.standard_normal((m, H)).astype(np.float32)
        x[4, 50] = np.nan
        logits = rng.standard_normal((m, E)).astype(np.float32)
        logits[0], logits[1, 1:], logits[2, :3] = -np.inf, -np.inf, np.nan
        kw = dict(k=4, n_group=1, topk_group=1, group_top=2, renorm=True, factor=1.0)
        rid, rw, rn = i8ref.route(logits, bias=None, score="softmax", **kw)
        assert rn.tolist() == [0, 1, 3, 4, 4]
        ids = np.concatenate((rid, np.tile(np.arange(E, E + shared), (m, 1))), 1)
        share = np.concatenate((rw, np.ones((m, shared))), 1)
        y = host(trmoe.moe_mx4(L, dev(x), rlog=dev(logits), score="softmax", **kw))
        want, tol = R.layer(x[:4].astype(np.float64), w["gate"], w["up"], w["down"], ids, share, "f32")
        within(y[:4], want, tol)
        assert np.isnan(y[4]).all()
        with pytest.raises(trmoe.TrkError, match="rlog"):
            trmoe.moe_mx4(L, dev(x), score="softmax", **kw)


def test_layer_poison_in_the_weights():
    """A scale byte of 255 in one expert's down row is that row's NaN, in its gate row all of its output's, for the tokens that
    choose it; rows and scales behind the stack's last are not looked at."""
    say("moe_mx4 poisoned weights")
    rng = np.random.default_rng(13)
    m, E, k, H, F = 6, 12, 3, 200, 70
    x, logits = rng.standard_normal((m, H)).astype(np.float32), rng.permutation(m * E).reshape(m, E).astype(np.float32) / (m * E)
    kw = dict(k=k, rlog=dev(logits), score="sigmoid")
    L, _, _, _, _ = layer_of(rng, E, H, F, router=False)
    clean = host(trmoe.moe_mx4(L, dev(x), **kw))
    e = int(np.argmax(logits[2]))
    chosen = np.array([e in np.argsort(-logits[t])[:k] for t in range(m)])
    assert chosen.any() and not chosen.all() and np.isfinite(clean).all()
    L.down.scale[e, 37, 2] = 255
    y = host(trmoe.moe_mx4(L, dev(x), **kw))
    assert np.isnan(y[chosen, 37]).all() and np.isnan(y).sum() == chosen.sum()
    assert np.array_equal(np.delete(y, 37, 1), np.delete(clean, 37, 1))
    L.gate.scale[e, 69, 6] = 255
    y = host(trmoe.moe_mx4(L, dev(x), **kw))
    assert np.isnan(y[chosen]).all() and np.array_equal(y[~chosen], clean[~chosen])


@pytest.mark.parametrize("m", [3, 8])
def test_work_of_any_content(m):
    """Memory that is given is used whatever it holds, and refused where it is too small; x may be the output."""
    import torch
    say(f"mx4 calls on given work, m={m}")
    rng = np.random.default_rng(14)
    E, k, H, F = 20, 5, 1100, 300
    L, _, _, _, _ = layer_of(rng, E, H, F, n_shared=1, gated=True)
    x = dev(rng.standard_normal((m, H)).astype(np.float32))
    want = trmoe.moe_mx4(L, x, k)
    n = L.work_values(k, m)
    for fill in (float("nan"), 1e38, 0.0):
        work = torch.full((n,), fill, device="cuda")
        assert torch.equal(trmoe.moe_mx4(L, x, k, work=work), want)
        assert torch.equal(trmoe.moe_mx4(L, x, k, work=work), want)
    for small in (work[:-1], work.double(), torch.empty((n, 2), device="cuda")[:, 0]):
        with pytest.raises(trmoe.TrkError, match="work"):
            trmoe.moe_mx4(L, x, k, work=small)
    assert torch.equal(trmoe.moe_mx4(L, x, k, out=x, work=work), want)
    big = dev(rng.standard_normal((40, H)).astype(np.float32))
    ids, w, ns = trmoe.route_scores((big @ L.router.T).contiguous(), k)
    plan = trmoe.experts_plan(ids, ns, k, E + 1)
    hq, hs = trmoe.quantize_mx4(trmoe.experts_up_mx4(L.gate, L.up, *trmoe.quantize_mx4(big), ids, ns, k, plan=plan))
    y = trmoe.experts_down_mx4(L.down, hq, hs, ids, w, ns, k, plan=plan)
    work = torch.full((40 * k * H,), float("nan"), device="cuda")
    assert torch.equal(trmoe.experts_down_mx4(L.down, hq, hs, ids, w, ns, k, plan=plan, work=work), y)
    with pytest.raises(trmoe.TrkError, match="work"):
        trmoe.experts_down_mx4(L.down, hq, hs, ids, w, ns, k, plan=plan, work=work[:-4])


# ---- together ----------------------------------------------------------------------------------------

def test_layer_is_the_calls_one_by_one():
    """The layer against routing, quantised rows and products of the same weights: the same up to the rows' quantisation."""
    import torch
    say("moe_mx4 against the calls one by one")
    rng = np.random.default_rng(4)
    m, E, k, H, F = 6, 32, 4, 512, 256
    L, w, r, _, _ = layer_of(rng, E, H, F)
    x = dev(rng.standard_normal((m, H)).astype(np.float32))
    logits = x @ L.router.T
    # rows that 4 bits hold: the layer and the calls then multiply the same values
    q, s = trmoe.quantize_mx4(x)
    xq = trmoe.dequantize_mx4(q, s, H)
    ids, wt, n = trmoe.route_scores(logits.contiguous(), k)
    h = trmoe.experts_up_mx4(L.gate, L.up, q, s, ids, n, k)
    x64 = host(xq).astype(np.float64)
    y = trmoe.moe_mx4(L, xq, k, rlog=logits.contiguous())
    want, tol = R.layer(x64, w["gate"], w["up"], w["down"], host(ids)[:, :k], host(wt)[:, :k].astype(np.float64), "f32")
    within(host(y), want, tol)
    hq, hs = trmoe.quantize_mx4(h)
    y2 = host(trmoe.experts_down_mx4(L.down, hq, hs, ids, wt, n, k))
    rel = np.linalg.norm(y2 - want) / np.linalg.norm(want)
    assert rel < 2 ** -2  # a 4-bit value is within 1/4 of its magnitude, a value below its block's least within that


def block(L, x, ids, w, n, slots, plan=None):
    q, s = trmoe.quantize_mx4(x)
    plan = trmoe.experts_plan(ids, n, slots, L.gate.count)
    h = trmoe.experts_up_mx4(L.gate, L.up, q, s, ids, n, slots, plan=plan, out=None, dtype=x.dtype)
    hq, hs = trmoe.quantize_mx4(h)
    return trmoe.experts_down_mx4(L.down, hq, hs, ids, w, n, slots, plan=plan, dtype=x.dtype)


@pytest.mark.parametrize("m", [5, 200])
def test_captured_and_replayed(m):
    """A block of the calls, and the layer, in a graph: every replay gives what the eager calls give on the same inputs."""
    import torch
    say(f"mx4 calls captured, m={m}")
    rng = np.random.default_rng(8)
    E, k, H, F = 16, 4, 320, 160
    L, _, _, _, _ = layer_of(rng, E, H, F, n_shared=1, gated=True)
    few = trmoe.MX4Layer(L.gate, L.up, L.down, router=L.router, n_shared=1, shared_gate=L.shared_gate)
    x = dev(rng.standard_normal((m, H)).astype(np.float32))
    W = trmoe.MX4Weights(*[t[0] for t in (L.gate.q, L.gate.scale)], H)

    def step():
        ids, w, n = trmoe.route_scores((x @ L.router.T).contiguous(), k)
        q, s = trmoe.quantize_mx4(x)
        return (block(L, x, ids, w, n, k), trmoe.gemm_mx4(W, q, s), trmoe.dequantize_mx4(q, s, H), trmoe.moe_mx4(few, x[:8], k))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for i in range(4):
        x.copy_(dev(rng.standard_normal((m, H)).astype(np.float32)))
        g.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_on_two_streams_at_once():
    import torch
    say("mx4 calls on two streams")
    rng = np.random.default_rng(9)
    E, k, H, F, m = 8, 2, 256, 128, 100
    L, _, _, _, _ = layer_of(rng, E, H, F)
    xs = [dev(rng.standard_normal((m, H)).astype(np.float32)) for _ in range(2)]
    routes = [trmoe.route_scores((x @ L.router.T).contiguous(), k) for x in xs]

    def both(x, r):
        return block(L, x, r[0], r[1], r[2], k), trmoe.moe_mx4(L, x[:8], k)
    want = [both(x, r) for x, r in zip(xs, routes)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for st, x, r in zip(streams, xs, routes):
            with torch.cuda.stream(st):
                got.append(both(x, r))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_a_stream_given():
    import torch
    say("mx4 calls on a given stream")
    rng = np.random.default_rng(10)
    E, k, H, F, m = 8, 2, 256, 128, 100
    L, _, _, _, _ = layer_of(rng, E, H, F)
    x = dev(rng.standard_normal((m, H)).astype(np.float32))
    ids, w, n = trmoe.route_scores((x @ L.router.T).contiguous(), k)
    want = block(L, x, ids, w, n, k), trmoe.moe_mx4(L, x[:8], k)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    q, s = trmoe.quantize_mx4(x, stream=st)
    plan = trmoe.experts_plan(ids, n, k, E, stream=st)
    h = trmoe.experts_up_mx4(L.gate, L.up, q, s, ids, n, k, plan=plan, stream=st)
    hq, hs = trmoe.quantize_mx4(h, stream=st)
    y = trmoe.experts_down_mx4(L.down, hq, hs, ids, w, n, k, plan=plan, stream=st)
    few = trmoe.moe_mx4(L, x[:8], k, stream=st)
    wide = torch.randn((2, 4, 6, 33), device="cuda")[:, :, :, ::1]
    W = trmoe.quantize_weights_mx4(wide[:, 1], stream=st)
    st.synchronize()
    assert torch.equal(y, want[0]) and torch.equal(few, want[1])
    codes, scale = R.quantize(host(wide[:, 1]).reshape(-1, 33))
    assert np.array_equal(host(W.q).reshape(-1, 32), R.pack(codes)) and np.array_equal(host(W.scale).reshape(-1, 2), scale)


@pytest.mark.parametrize("m", [3, 150])
def test_the_same_bits_every_time(m):
    import torch
    say(f"mx4 calls repeated, m={m}")
    rng = np.random.default_rng(11)
    E, k, H, F = 8, 4, 512, 256
    L, _, _, _, _ = layer_of(rng, E, H, F)
    x = dev(rng.standard_normal((m, H)).astype(np.float32))
    ids, w, n = trmoe.route_scores((x @ L.router.T).contiguous(), k)
    first = block(L, x, ids, w, n, k)
    for _ in range(5):
        assert torch.equal(block(L, x, ids, w, n, k), first)
        if m <= 8:
            assert torch.equal(trmoe.moe_mx4(L, x, k), trmoe.moe_mx4(L, x, k))


def test_empty_batches():
    import torch
    say("mx4 calls of no rows")
    rng = np.random.default_rng(12)
    L, _, _, _, _ = layer_of(rng, 4, 64, 32)
    x = torch.zeros((0, 64), device="cuda")
    q, s = trmoe.quantize_mx4(x)
    assert q.shape == (0, 32) and s.shape == (0, 2) and trmoe.dequantize_mx4(q, s, 64).shape == (0, 64)
    assert trmoe.gemm_mx4(trmoe.MX4Weights(L.gate.q[0], L.gate.scale[0], 64), q, s).shape == (0, 32)
    assert trmoe.moe_mx4(L, x, 2).shape == (0, 64)
    with pytest.raises(trmoe.TrkError, match="above 8"):
        trmoe.moe_mx4(L, torch.zeros((9, 64), device="cuda"), 2)


def test_a_stream_of_another_device():
    """Every call refuses it, and takes one of its own."""
    import torch
    from types import SimpleNamespace
    say("mx4 calls: streams of another device")
    there = SimpleNamespace(cuda_stream=0, device_index=torch.cuda.current_device() + 1)
    W = trmoe.quantize_weights_mx4(torch.randn((4, 32, 32), device="cuda"))
    x = torch.randn((40, 32), device="cuda")
    q, s = trmoe.quantize_mx4(x)
    ids, w, n = trmoe.route_scores(torch.randn((40, 4), device="cuda"), 2)
    plan = trmoe.experts_plan(ids, n, 2, 4)
    hq, hs = trmoe.quantize_mx4(trmoe.experts_up_mx4(W, W, q, s, ids, n, 2, plan=plan))
    L = trmoe.MX4Layer(W, W, W, router=torch.randn((4, 32), device="cuda"))
    y, h = torch.full((40, 32), 9.0, device="cuda"), torch.full((80, 32), 9.0, device="cuda")
    work, few = torch.empty(40 * 2 * 32, device="cuda"), torch.empty(L.work_values(2, 8), device="cuda")
    one = trmoe.MX4Weights(W.q[0], W.scale[0], 32)
    for call in (lambda st: trmoe.quantize_mx4(x, out=(q.clone(), torch.empty((40, 4), dtype=torch.uint8, device="cuda")[:, :1]), stream=st),
                 lambda st: trmoe.dequantize_mx4(q, s, 32, out=y, stream=st),
                 lambda st: trmoe.gemm_mx4(one, q, s, out=y, stream=st),
                 lambda st: trmoe.experts_up_mx4(W, W, q, s, ids, n, 2, plan=plan, out=h, stream=st),
                 lambda st: trmoe.experts_down_mx4(W, hq, hs, ids, w, n, 2, plan=plan, out=y, work=work, stream=st),
                 lambda st: trmoe.moe_mx4(L, x[:8], 2, out=y[:8], work=few, stream=st)):
        with pytest.raises(trmoe.TrkError, match="a stream of device"):
            call(there)
        call(torch.cuda.current_stream())
    torch.cuda.synchronize()


def test_the_layer_captured_with_a_launch_for_the_choice():
    import torch
    say("moe_mx4 captured, the choice apart")
    rng = np.random.default_rng(15)
    m, E, k, H, F = 8, 24, 6, 1100, 700
    L, _, _, _, _ = layer_of(rng, E, H, F, n_shared=1)
    x = dev(rng.standard_normal((m, H)).astype(np.float32))
    work = torch.empty(L.work_values(k, m), device="cuda")
    trmoe.moe_mx4(L, x, k, work=work)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = trmoe.moe_mx4(L, x, k, work=work)
        y2 = trmoe.moe_mx4(L, y, k, work=work)  # one after another on the same work
    for _ in range(3):
        x.copy_(dev(rng.standard_normal((m, H)).astype(np.float32)))
        g.replay()
        torch.cuda.synchronize()
        a, b = y.clone(), y2.clone()
        assert torch.equal(trmoe.moe_mx4(L, x, k), a) and torch.equal(trmoe.moe_mx4(L, a, k), b)
        torch.cuda.synchronize()
