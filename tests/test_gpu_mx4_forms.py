"""Every kernel of the 4-bit products at sizes that the rules send to it (tests/mx4forms.py), against 64-bit forms: 16- and 32-bit
outputs, a bias, an output that is added to, an item of a stack, scales of NaN, rows too far apart for tiles."""
from __future__ import annotations

import i8ref
import mx4forms as S
import mx4ref as R
import numpy as np
import pytest

import trmoe
from test_gpu_mx4 import DTYPES, apart, dev, host, routing, rows4, say

pytestmark = pytest.mark.gpu


def rounded(y, dtype):
    """What rounding y (float64, on the GPU) to `dtype` may move it by."""
    return i8ref.EPS[dtype] * y.abs() + i8ref.LEAST[dtype]


def gemm_tol(mag, k, want, dtype, *added):
    """mx4ref.gemm_tol on the GPU: the sum's steps, one rounding to 32 bits for each term added, the output's."""
    a, err = want.abs(), (R.blocks(k) + 8) * R.STEP * mag
    for more in added:
        a = a + more.abs()
        err = err + 1.01 * i8ref.EPS["f32"] * a
    return err + 1.01 * rounded(a, dtype)


def inside(got, want, tol):
    assert got.isfinite().all()
    far = ((got.double() - want).abs() / tol).max().item()
    assert far <= 1, far


GEMMS = [(form, *size) for form, sizes in S.GEMMS.items() for size in sizes]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form,m,rows,k", GEMMS)
def test_gemm_of_each_form(form, m, rows, k, dtype):
    import torch
    say(f"gemm_mx4 {form} {m} x {rows} x {k} {dtype}")
    rng = np.random.default_rng(m + rows + k)
    (q, s), (wq, ws) = rows4(rng, m, k), rows4(rng, rows, k)
    xd, to = apart(q, s, 2), i8ref.torch_dtype(dtype)
    stack = [torch.stack((t.roll(1, 0), t)) for t in apart(wq, ws)]  # the second of two, the first something else
    wide = [torch.full((*t.shape[:-1], (t.shape[-1] + 15) // 16 * 16 + 16), 255, dtype=torch.uint8, device="cuda") for t in stack]
    for w, t in zip(wide, stack):
        w[..., :t.shape[-1]] = t
    W = trmoe.MX4Weights(*[w[..., :t.shape[-1]] for w, t in zip(wide, stack)], k)
    x, w = dev(R.values(q, s, k)), dev(R.values(wq, ws, k))
    want, mag = x @ w.T, x.abs() @ w.abs().T
    bias = dev(rng.standard_normal(rows).astype(np.float32))
    y = trmoe.gemm_mx4(W, *xd, bias=bias, dtype=to, item=1)
    b = bias.double()[None, :]
    inside(y, want + b, gemm_tol(mag, k, want, dtype, b))
    # added to, in a slice of a wider output
    out = torch.randn((m, rows + 5), device="cuda").to(to)
    before = out.clone()
    trmoe.gemm_mx4(W, *xd, out=out[:, 1:1 + rows], accumulate=True, item=1)
    old = before[:, 1:1 + rows].double()
    inside(out[:, 1:1 + rows], want + old, gemm_tol(mag, k, want, dtype, old))
    assert torch.equal(out[:, 0], before[:, 0]) and torch.equal(out[:, 1 + rows:], before[:, 1 + rows:])
    # a NaN scale in the last row of each, in the last and in the first block
    xd[1][m - 1, R.blocks(k) - 1], W.scale[1, rows - 1, 0] = 255, 255
    z = trmoe.gemm_mx4(W, *xd, bias=bias, dtype=to, item=1)
    nan = torch.zeros((m, rows), dtype=torch.bool, device="cuda")
    nan[m - 1], nan[:, rows - 1] = True, True
    assert torch.equal(z.isnan(), nan) and torch.equal(z[~nan], y[~nan])


def entries_of(there, ids, slots, E):
    for e in range(E):
        t, j = np.nonzero(there & (ids[:, :slots] == e))
        if t.size:
            yield e, dev(t), dev(j)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", list(S.UP))
def test_up_of_each_form(form, dtype):
    import torch
    m, slots, E, F = S.UP[form]
    k, to = 1100, i8ref.torch_dtype(dtype)
    say(f"experts_up_mx4 {form} m={m} slots={slots} E={E} F={F} {dtype}")
    rng = np.random.default_rng(m + E + F)
    (q, s), (gq, gs), (uq, us) = rows4(rng, m, k), rows4(rng, E, F, k, spread=k ** -0.5), rows4(rng, E, F, k, spread=k ** -0.5)
    ids, w, n = routing(rng, m, E, slots, "ragged" if E > 20 else "one")
    idt, nt = dev(ids), dev(n)
    xd, G, U = apart(q, s), trmoe.MX4Weights(*apart(gq, gs), k), trmoe.MX4Weights(*apart(uq, us, 2), k)
    plan = trmoe.experts_plan(idt, nt, slots, E)
    out = torch.full((m * slots, F + 2), 9.0, dtype=to, device="cuda")
    trmoe.experts_up_mx4(G, U, *xd, idt, nt, slots, plan=plan, out=out[:, 1:1 + F])
    there = i8ref.entries(ids, n, slots, E)
    none = dev(~there.reshape(-1))
    assert (out[:, 0] == 9).all() and (out[:, 1 + F:] == 9).all() and (out[none] == 9).all()
    h, x = out[:, 1:1 + F], dev(R.values(q, s, k))
    steps = (R.blocks(k) + 8) * R.STEP
    for e, t, j in entries_of(there, ids, slots, E):
        ge, ue = dev(R.values(gq[e], gs[e], k)), dev(R.values(uq[e], us[e], k))
        g, u = x[t] @ ge.T, x[t] @ ue.T
        eg, eu = steps * (x[t].abs() @ ge.abs().T), steps * (x[t].abs() @ ue.abs().T)
        silu = g * torch.sigmoid(g)
        hm = silu.abs() * u.abs()
        # mx4ref.swiglu_tol
        tol = 1.1 * eg * u.abs() + silu.abs() * eu + 1.1 * eg * eu + 8.1 * i8ref.EPS["f32"] * hm + 1.01 * rounded(hm, dtype)
        inside(h[t * slots + j], silu * u, tol)
    # a NaN scale in a token's row, and in an expert's last row of up
    hit = np.zeros((m * slots, F), bool)
    tp = int(np.nonzero(there.any(1))[0][-1])
    ep = int(ids[np.nonzero(there[:, 0])[0][0], 0])
    xd[1][tp, R.blocks(k) - 1], U.scale[ep, F - 1, 0] = 255, 255
    hit[tp * slots:(tp + 1) * slots] = there[tp][:, None]
    hit[(there & (ids[:, :slots] == ep)).reshape(-1), F - 1] = True
    again = torch.full((m * slots, F), 9.0, dtype=to, device="cuda")
    trmoe.experts_up_mx4(G, U, *xd, idt, nt, slots, plan=plan, out=again)
    hit = dev(hit)
    assert torch.equal(again.isnan(), hit) and torch.equal(again[~hit], h[~hit])


@pytest.mark.parametrize("form,dtype", [(form, DTYPES[i % 3]) for i, form in enumerate(S.DOWN)])
def test_down_of_each_form(form, dtype):
    import torch
    m, slots, E, H = S.DOWN[form]
    k, to = 1100, i8ref.torch_dtype(dtype)
    say(f"experts_down_mx4 {form} m={m} slots={slots} E={E} H={H} {dtype}")
    rng = np.random.default_rng(m + E + H)
    (q, s), (wq, ws) = rows4(rng, m * slots, k), rows4(rng, E, H, k)
    ids, wt, n = routing(rng, m, E, slots, "ragged" if E > 20 else "one")
    idt, nt, wd = dev(ids), dev(n), dev(wt)
    qs, W = apart(q, s), trmoe.MX4Weights(*apart(wq, ws), k)
    plan = trmoe.experts_plan(idt, nt, slots, E)
    y = trmoe.experts_down_mx4(W, *qs, idt, wd, nt, slots, plan=plan, dtype=to)
    there = i8ref.entries(ids, n, slots, E)
    x = dev(R.values(q, s, k))
    want, tol, mag = [torch.zeros((m, H), dtype=torch.float64, device="cuda") for _ in range(3)]
    for e, t, j in entries_of(there, ids, slots, E):
        de, share = dev(R.values(wq[e], ws[e], k)), wd[t, j].double()[:, None]
        v, a = x[t * slots + j] @ de.T * share, x[t * slots + j].abs() @ de.abs().T * share
        want.index_put_((t,), v, accumulate=True), mag.index_put_((t,), v.abs(), accumulate=True)
        tol.index_put_((t,), (R.blocks(k) + 8) * R.STEP * a, accumulate=True)
    # a weight's product and each sum of the slots round once
    tol = tol + (slots + 2) * i8ref.EPS["f32"] * mag
    inside(y, want, tol + 1.01 * rounded(mag + tol, dtype))
    added = y.clone()
    trmoe.experts_down_mx4(W, *qs, idt, wd, nt, slots, plan=plan, out=added, accumulate=True)
    both = mag + y.double().abs()
    inside(added, want + y.double(), tol + 1.01 * i8ref.EPS["f32"] * both + 1.01 * rounded(both + tol, dtype))
    # a NaN scale in an entry's row, and in an expert's last row
    hit = np.zeros((m, H), bool)
    tp = int(np.nonzero(there[:, 0])[0][-1])
    ep = int(ids[np.nonzero(there[:, 0])[0][0], 0])
    qs[1][tp * slots, R.blocks(k) - 1], W.scale[ep, H - 1, 0] = 255, 255
    hit[tp] = True
    hit[(there & (ids[:, :slots] == ep)).any(1), H - 1] = True
    again = trmoe.experts_down_mx4(W, *qs, idt, wd, nt, slots, plan=plan, dtype=to)
    hit = dev(hit)
    assert torch.equal(again.isnan(), hit) and torch.equal(again[~hit], y[~hit])


@pytest.mark.parametrize("H", [1, 2, 3, 4, 5, 6, 7, 1021, 1022, 1023, 1026])
@pytest.mark.parametrize("bits", [4, 8])
def test_down_of_any_number_of_columns(bits, H):
    """The sum over a token's entries, four columns at a time, in slot order: as numpy adds the same 32-bit rows."""
    import torch
    say(f"experts_down bits={bits} H={H}")
    rng = np.random.default_rng(H)
    m, E, slots, k = 30, 6, 5, 64
    ids, wt, n = routing(rng, m, E, slots, "ragged")
    idt, nt, wd = dev(ids), dev(n), dev(wt)
    plan = trmoe.experts_plan(idt, nt, slots, E)
    x, w = [dev(rng.standard_normal(s).astype(np.float32)) for s in ((m * slots, k), (E, H, k))]
    if bits == 4:
        q, W, down = trmoe.quantize_mx4(x), trmoe.quantize_weights_mx4(w), trmoe.experts_down_mx4
    else:
        q, W, down = trmoe.quantize_rows(x), trmoe.quantize_weights(w), trmoe.experts_down_i8
    work = torch.full((m * slots * H + 64,), float("nan"), device="cuda")
    old = torch.randn((m, H + 3), device="cuda")
    y = old.clone()
    down(W, *q, idt, wd, nt, slots, plan=plan, out=y[:, 1:1 + H], work=work, accumulate=True)
    rows = host(work)[:m * slots * H].reshape(m, slots, H)  # the entries' weighted rows
    there = i8ref.entries(ids, n, slots, E)
    assert np.isfinite(rows[there]).all() and (np.abs(rows[there]).max(1) > 0).all() and work[m * slots * H:].isnan().all()
    want = np.zeros((m, H), np.float32)
    for j in range(slots):
        want = np.where(there[:, j:j + 1], want + rows[:, j], want)
    assert np.array_equal(host(y)[:, 1:1 + H], want + host(old)[:, 1:1 + H])
    assert torch.equal(y[:, 0], old[:, 0]) and torch.equal(y[:, 1 + H:], old[:, 1 + H:])


# ---- rows too far apart for the tiles' 32-bit offsets ---------------------------------------------------

def far_rows(t, ld):
    """The same rows, ld bytes apart."""
    import torch
    rows = t.shape[-2]
    far = torch.empty((*t.shape[:-2], rows, ld), dtype=torch.uint8, device="cuda")[..., :t.shape[-1]]
    far.copy_(t)
    return far


@pytest.mark.parametrize("what", ["x", "x scales", "w", "w scales"])
def test_gemm_of_rows_far_apart(what):
    say(f"gemm_mx4 rows far apart: {what}")
    m, rows, k = S.FAR_X if what[0] == "x" else S.FAR_W
    rng = np.random.default_rng(m)
    (q, s), (wq, ws) = rows4(rng, m, k), rows4(rng, rows, k)
    xs, W = list(apart(q, s)), list(apart(wq, ws))
    of, i = (xs if what[0] == "x" else W), (1 if "scales" in what else 0)
    of[i] = far_rows(of[i], 1 << 23)
    y = trmoe.gemm_mx4(trmoe.MX4Weights(*W, k), *xs)
    x, w = dev(R.values(q, s, k)), dev(R.values(wq, ws, k))
    want = x @ w.T
    inside(y, want, gemm_tol(x.abs() @ w.abs().T, k, want, "f32"))


@pytest.mark.parametrize("what", ["x", "x scales", "w", "w scales"])
@pytest.mark.parametrize("call", ["up", "down"])
def test_experts_of_rows_far_apart(call, what):
    """Each planned call then takes its entries one by one."""
    import torch
    say(f"experts_{call}_mx4 rows far apart: {what}")
    rng = np.random.default_rng(6)
    m, E, slots, k, rows = 40, 3, 2, 96, 40
    n_x = m if call == "up" else m * slots
    (q, s), (wq, ws), (uq, us) = rows4(rng, n_x, k), rows4(rng, E, rows, k), rows4(rng, E, rows, k)
    ids, wt, n = routing(rng, m, E, slots, "ragged")
    idt, nt, wd = dev(ids), dev(n), dev(wt)
    xs, W = list(apart(q, s)), list(apart(wq, ws))
    of, i = (xs if what[0] == "x" else W), (1 if "scales" in what else 0)
    ld = 1 << 23 if what[0] == "w" else (1 << 32) // n_x // 16 * 16 + 16
    of[i] = far_rows(of[i], ld)
    G, U = trmoe.MX4Weights(*W, k), trmoe.MX4Weights(*apart(uq, us), k)
    plan = trmoe.experts_plan(idt, nt, slots, E)
    there = i8ref.entries(ids, n, slots, E)
    x, g64 = R.values(q, s, k), R.values(wq, ws, k)
    if call == "up":
        h = torch.full((m * slots, rows), 9.0, device="cuda")
        trmoe.experts_up_mx4(G, U, *xs, idt, nt, slots, plan=plan, out=h)
        u64, got = R.values(uq, us, k), host(h)
        assert (got[~there.reshape(-1)] == 9).all()
        for t, j in zip(*np.nonzero(there)):
            e = ids[t, j]
            xt = x[t:t + 1]
            g, u = xt @ g64[e].T, xt @ u64[e].T
            tol = R.swiglu_tol(g, u, R.sum_tol(xt, g64[e]), R.sum_tol(xt, u64[e]), "f32")
            assert (np.abs(got[t * slots + j] - R.silu(g) * u) <= tol).all()
        return
    y = host(trmoe.experts_down_mx4(G, *xs, idt, wd, nt, slots, plan=plan))
    want, tol, mag = np.zeros((m, rows)), np.zeros((m, rows)), np.zeros((m, rows))
    for t, j in zip(*np.nonzero(there)):
        xt, de, share = x[t * slots + j][None], g64[ids[t, j]], float(wt[t, j])
        v = (xt @ de.T)[0] * share
        want[t] += v
        mag[t] += np.abs(v)
        tol[t] += R.sum_tol(xt, de)[0] * share
    tol = tol + (slots + 2) * i8ref.EPS["f32"] * mag
    assert (np.abs(y - want) <= tol + 1.01 * i8ref.round_rel(mag + tol, "f32")).all()
    assert (y[~there.any(1)] == 0).all()


# ---- shared experts --------------------------------------------------------------------------------------

@pytest.mark.parametrize("m", [5, 200])
def test_shared_experts_as_further_entries(m):
    """A shared expert behind each token's chosen ones, also where those are fewer than k: the same up and down calls."""
    import torch
    say(f"mx4 calls with shared experts as entries, m={m}")
    rng = np.random.default_rng(m)
    E, k, H, F = 12, 3, 320, 200
    w = {"gate": rows4(rng, E + 1, F, H, spread=H ** -0.5), "up": rows4(rng, E + 1, F, H, spread=H ** -0.5), "down": rows4(rng, E + 1, H, F)}
    size = {"gate": H, "up": H, "down": F}
    gate, up, down = [trmoe.MX4Weights(*apart(*w[i]), size[i]) for i in w]
    v = {i: R.values(*w[i], size[i]) for i in w}
    x = dev(rng.standard_normal((m, H)).astype(np.float32))
    logits = dev(rng.standard_normal((m, E)).astype(np.float32))
    logits[0], logits[1, 2:] = -np.inf, -np.inf  # none and two of them
    share = dev(rng.uniform(0.1, 0.9, (m, 1)).astype(np.float32))
    ids, wt, n = trmoe.route_scores(logits, k, score="softmax")
    at = n.long()[:, None]
    ids.scatter_(1, at, E), wt.scatter_(1, at, share), n.add_(1)
    assert host(n)[:2].tolist() == [1, 3] and (host(n)[2:] == k + 1).all()
    plan = trmoe.experts_plan(ids, n, k + 1, E + 1)
    q, s = trmoe.quantize_mx4(x)
    h = torch.zeros((m * (k + 1), F), device="cuda")
    trmoe.experts_up_mx4(gate, up, q, s, ids, n, k + 1, plan=plan, out=h)
    hq, hs = trmoe.quantize_mx4(h)
    y = host(trmoe.experts_down_mx4(down, hq, hs, ids, wt, n, k + 1, plan=plan))
    x64, h64 = R.values(host(q), host(s), H), R.values(host(hq), host(hs), F)
    ids, wt, n, h = host(ids), host(wt).astype(np.float64), host(n), host(h)
    for t in range(m):
        want, tol, mag = np.zeros(H), np.zeros(H), np.zeros(H)
        for j in range(n[t]):
            e, xt, ht = ids[t, j], x64[t:t + 1], h64[t * (k + 1) + j][None]
            assert (e == E) == (j == n[t] - 1)
            g, u = xt @ v["gate"][e].T, xt @ v["up"][e].T
            off = R.swiglu_tol(g, u, R.sum_tol(xt, v["gate"][e]), R.sum_tol(xt, v["up"][e]), "f32")
            assert (np.abs(h[t * (k + 1) + j] - R.silu(g) * u) <= off).all()
            a = (ht @ v["down"][e].T)[0] * wt[t, j]
            want, mag, tol = want + a, mag + np.abs(a), tol + R.sum_tol(ht, v["down"][e])[0] * wt[t, j]
        tol = tol + (k + 3) * i8ref.EPS["f32"] * mag
        assert (np.abs(y[t] - want) <= tol + 1.01 * i8ref.round_rel(mag + tol, "f32")).all()
