"""The int8 products and the quantisation of rows at the ends of their arguments, on the GPU against their plain 64-bit forms
(tests/i8ref.py)."""
from __future__ import annotations

import i8ref as R
import numpy as np
import pytest

import trmoe
from test_gpu_scores_i8 import dev, host, i8, padded, routing, say, scales

pytestmark = pytest.mark.gpu


def test_weights_of_a_wider_stack_on_a_stream():
    """Rows that make no one matrix are copied first: on the stream given, whatever the current one still has to do."""
    import torch
    say("quantize_weights of a slice, on a stream")
    E, rows, k = 16, 500, 1000
    wide = torch.randn((E, rows + 36, k), device="cuda")
    w = wide[:, :rows]
    want = trmoe.quantize_weights(w.contiguous())
    a, b = (torch.randn((4096, 4096), device="cuda") for _ in range(2))
    st = torch.cuda.Stream()
    for _ in range(3):
        st.wait_stream(torch.cuda.current_stream())
        for _ in range(20):
            torch.mm(a, a, out=b)  # nothing is freed here that the call could be given
        got = trmoe.quantize_weights(w, stream=st)
        junk = [torch.full((E * rows * k,), float("nan"), device="cuda") for _ in range(2)]  # over what was given back
        torch.cuda.synchronize()
        assert torch.equal(got.q, want.q) and torch.equal(got.scale, want.scale)
        del got, junk


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("k", [(1 << 32) - 5, (1 << 32) - (1 << 15)])
def test_quantize_the_longest_rows(dtype, k):
    """A row of nearly 2^32 values: places in it that 32 bits do not add up."""
    import torch
    say(f"quantize_rows {dtype} k={k}")
    part = 1 << 28
    # repeated at a length that divides no piece; the largest value far from both ends
    base = torch.arange(part, device="cuda").remainder_(509).sub_(254).to(R.torch_dtype(dtype))
    x = torch.empty((1, k), dtype=base.dtype, device="cuda")
    for at in range(0, k, part):
        x[0, at:at + part] = base[:k - at]
    x[0, 3 * part + 17] = 508
    q = torch.full((1, k + 16), 99, dtype=torch.int8, device="cuda")
    s = torch.empty(1, device="cuda")
    trmoe.quantize_rows(x, out=(q[:, :k], s))
    assert s.item() == np.float32(508 / 127)
    want = (base.double() / 4).round().to(torch.int8)  # 127 x / 508: whole quarters, ties to even
    for at in range(0, k, part):
        got = q[0, at:min(at + part, k)]
        if at == 3 * part:
            assert got[17] == 127
            got[17] = want[17]
        assert torch.equal(got, want[:got.numel()]), at
    assert (q[0, k:] == 99).all()


@pytest.mark.parametrize("far", ["weight rows", "tokens"])
def test_gemm_i8_of_the_most_rows(far):
    """2^32 - 256 - 3 rows on one side (64 GB at k = 16), one on the other: the last tile's numbers still fit 32 bits."""
    import torch
    say(f"gemm_i8 most {far}")
    n, k, part = (1 << 32) - 259, 16, 1 << 24
    gen = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randint(-127, 128, (part, k), dtype=torch.int8, device="cuda", generator=gen)
    one = torch.randint(-127, 128, (1, k), dtype=torch.int8, device="cuda", generator=gen)
    many = torch.empty((n, k), dtype=torch.int8, device="cuda")
    scale = torch.ones(n, device="cuda")
    for at in range(0, n, part):
        many[at:at + part] = base[:n - at]
        scale[at] = 2.0  # a mark at each part's head
    unit = torch.ones(1, device="cuda")
    if far == "tokens":
        y = torch.empty((n, 1), dtype=torch.float16, device="cuda")
        trmoe.gemm_i8(trmoe.I8Weights(one, unit), many, scale, out=y)
    else:
        y = torch.empty((1, n), dtype=torch.float16, device="cuda")
        trmoe.gemm_i8(trmoe.I8Weights(many, scale), one, unit, out=y)
    want = (base.double() @ one.double().t()).view(-1)  # whole numbers below 2^18
    want[0] *= 2
    want = want.half()
    y = y.view(-1)
    for at in range(0, n, part):
        assert torch.equal(y[at:at + part], want[:n - at]), at


# (m, slots, E) of the call, of the plan: as many words, other entries or experts
@pytest.mark.parametrize("call,made", [((199, 2, 64), (200, 2, 64)), ((200, 2, 64), (100, 4, 64)), ((10, 3, 64), (10, 3, 40)),
                                       ((10, 3, 64), (15, 2, 64)), ((1200, 4, 80), (2400, 2, 80)), ((40, 2, 16), None)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_a_plan_of_another_call(call, made, dtype):
    """A plan of as many words, made for other sizes, or none that was made: entries' rows of h, and of y the rows of tokens
    that have any, are NaN; the rest stays."""
    import torch
    say(f"experts {call} with the plan of {made} {dtype}")
    rng = np.random.default_rng(7)
    m, slots, E = call
    H, F = 96, 80
    ids, w, n = routing(rng, m, E, slots, "elsewhere")
    di, dw, dn = dev(ids), dev(w), dev(n)
    own = trmoe.experts_plan(di, dn, slots, E)
    if made:
        mi, _, mn = routing(rng, made[0], made[2], made[1], "plain")
        other = trmoe.experts_plan(dev(mi), dev(mn), made[1], made[2])
    else:
        other = torch.zeros_like(own)
    assert other.shape == own.shape
    gate, up = (trmoe.I8Weights(padded(i8(rng, E, F, H)), dev(scales(rng, E, F))) for _ in range(2))
    down = trmoe.I8Weights(padded(i8(rng, E, H, F)), dev(scales(rng, E, H)))
    q, s = dev(i8(rng, m, H)), dev(scales(rng, m))
    hq, hs = dev(i8(rng, m * slots, F)), dev(scales(rng, m * slots))
    live = R.entries(ids, n, slots, E)
    has, live = live.any(1), live.reshape(-1)
    assert has.any() and not has.all()
    for plan in (other, own):
        wide = torch.full((m * slots + 1, F + 3), 9.0, dtype=R.torch_dtype(dtype), device="cuda")
        trmoe.experts_up_i8(gate, up, q, s, di, dn, slots, plan=plan, out=wide[:m * slots, :F])
        h = host(wide)
        assert (h[:-1][~live] == 9).all() and (h[-1] == 9).all() and (h[:, F:] == 9).all()
        for acc in (False, True):
            wide = torch.full((m + 1, H + 3), 9.0, dtype=R.torch_dtype(dtype), device="cuda")
            trmoe.experts_down_i8(down, hq, hs, di, dw, dn, slots, plan=plan, out=wide[:m, :H], accumulate=acc)
            y = host(wide)
            assert (y[m] == 9).all() and (y[:, H:] == 9).all()
            assert np.isnan(y[:m, :H][has]).all() if plan is other else np.isfinite(y[:m, :H]).all()
            assert (y[:m, :H][~has] == (9 if acc else 0)).all()
        assert np.isnan(h[:-1, :F][live]).all() if plan is other else not np.isnan(h).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m", [1, 40])
def test_silu_of_far_gates(m, dtype):
    """Gates beyond the exponential's usual range: silu falls with it, down to the smallest numbers.  The exponential is
    within 2^-22 as nearer to zero, two roundings follow: less than swiglu_tol counts."""
    say(f"experts_up far gates m={m} {dtype}")
    rng = np.random.default_rng(m)
    G = np.concatenate([np.linspace(-130, -70, 241), [-1e3, -1e30, -300.0, 60.0, 200.0, 1e4, 0.0]])
    F, H = G.size, 16
    U = np.exp(rng.uniform(-10, 60 if dtype != "f16" else 5, F)) * rng.choice([-1, 1], F)
    U[np.abs(G) > 150] = 0.5
    q = np.zeros((m, H), np.int8)
    q[:, 3] = 127
    w = np.zeros((1, F, H), np.int8)
    w[0, :, 3] = 127
    gw, uw = w * np.where(G < 0, -1, 1).astype(np.int8)[None, :, None], w * np.where(U < 0, -1, 1).astype(np.int8)[None, :, None]
    gs, us = ((np.abs(a) / 127 ** 2).astype(np.float32)[None] for a in (G, U))
    s = np.ones(m, np.float32)
    ids, n = np.zeros((m, 32), np.int32), np.ones(m, np.int32)
    di, dn = dev(ids), dev(n)
    gate, up = trmoe.I8Weights(dev(gw), dev(gs)), trmoe.I8Weights(dev(uw), dev(us))
    got = host(trmoe.experts_up_i8(gate, up, dev(q), dev(s), di, dn, 1, plan=trmoe.experts_plan(di, dn, 1, 1),
                                   dtype=R.torch_dtype(dtype))).astype(np.float64)
    g, u = R.gemm(q, s, gw[0], gs[0]), R.gemm(q, s, uw[0], us[0])
    with np.errstate(over="ignore"):
        want, tol = R.swiglu(g, u), R.swiglu_tol(g, u, dtype)
    assert (np.abs(got - want) <= tol).all(), np.argwhere(~(np.abs(got - want) <= tol))[:4]


@pytest.mark.parametrize("m", [1, 40])
def test_silu_of_a_gate_out_of_range(m):
    """A gate product below the lowest number: nothing is left of its silu."""
    import torch
    say(f"experts_up gate out of range m={m}")
    one = torch.ones((1, 8, 16), dtype=torch.int8, device="cuda")
    gate = trmoe.I8Weights(-one, torch.full((1, 8), 3e38, device="cuda"))
    up = trmoe.I8Weights(one, torch.ones((1, 8), device="cuda"))
    ids, n = torch.zeros((m, 32), dtype=torch.int32, device="cuda"), torch.ones(m, dtype=torch.int32, device="cuda")
    h = trmoe.experts_up_i8(gate, up, one[0, :1].expand(m, 16).contiguous(), torch.ones(m, device="cuda"), ids, n, 1,
                            plan=trmoe.experts_plan(ids, n, 1, 1))
    assert (h == 0).all()


def test_a_stream_of_another_device():
    """Every call refuses it, and takes one of its own."""
    import torch
    from types import SimpleNamespace
    say("streams of another device")
    there = SimpleNamespace(cuda_stream=0, device_index=torch.cuda.current_device() + 1)
    W = trmoe.quantize_weights(torch.randn((4, 32, 32), device="cuda"))
    x = torch.randn((40, 32), device="cuda")
    q, s = trmoe.quantize_rows(x)
    ids, w, n = trmoe.route_scores(torch.randn((40, 4), device="cuda"), 2)
    plan = trmoe.experts_plan(ids, n, 2, 4)
    hq, hs = trmoe.quantize_rows(trmoe.experts_up_i8(W, W, q, s, ids, n, 2, plan=plan))
    y, h = torch.full((40, 32), 9.0, device="cuda"), torch.full((80, 32), 9.0, device="cuda")
    work = torch.empty(40 * 2 * 32, device="cuda")
    for call in (lambda st: trmoe.quantize_rows(x, out=(hq[:40].clone(), s.clone()), stream=st),
                 lambda st: trmoe.route_scores(x, 2, stream=st),
                 lambda st: trmoe.gemm_i8(trmoe.I8Weights(W.q[0], W.scale[0]), q, s, out=y, stream=st),
                 lambda st: trmoe.experts_plan(ids, n, 2, 4, stream=st),
                 lambda st: trmoe.experts_up_i8(W, W, q, s, ids, n, 2, plan=plan, out=h, stream=st),
                 lambda st: trmoe.experts_down_i8(W, hq, hs, ids, w, n, 2, plan=plan, out=y, work=work, stream=st)):
        with pytest.raises(trmoe.TrkError, match="a stream of device"):
            call(there)
        call(torch.cuda.current_stream())
    torch.cuda.synchronize()
