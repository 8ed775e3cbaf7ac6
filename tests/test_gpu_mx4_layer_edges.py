"""The layer on 4-bit experts where its activations are no numbers or nearly too large, and where its choice takes 64 bits."""
from __future__ import annotations

import i8ref
import mx4ref as R
import numpy as np
import pytest

import trmoe
from test_gpu_mx4 import apart, dev, host, layer_of, rows4, say, within

pytestmark = pytest.mark.gpu


# (m, F): the choice by every workgroup of gate and up, and by a launch of its own
CHOICES = [(6, 70), (8, 1100)]


@pytest.mark.parametrize("score,bias", [("sigmoid", True), ("softmax", False), ("softmax", True)])
@pytest.mark.parametrize("shared", [0, 1])
@pytest.mark.parametrize("m,F", CHOICES)
def test_a_poisoned_token_through_the_router(m, F, shared, score, bias):
    """A NaN or an infinity in x makes the token's own row NaN, also where its logits are such that no expert is chosen."""
    say(f"moe_mx4 poisoned tokens m={m} F={F} shared={shared} {score} bias={bias}")
    rng = np.random.default_rng(m + F)
    E, k, H = 12, 4, 1100
    L, _, _, _, _ = layer_of(rng, E, H, F, n_shared=shared, bias=bias)
    x = rng.standard_normal((m, H)).astype(np.float32)
    for dtype in ("f32", "bf16", "f16"):
        clean = dev(x).to(i8ref.torch_dtype(dtype))
        want = host(trmoe.moe_mx4(L, clean, k, score=score))
        assert np.isfinite(want).all()
        for places in ([(1, 0, np.nan), (3, 1099, np.inf), (5, 500, -np.inf)], [(0, 31, -np.inf), (4, 1023, np.nan)],
                       [(2, 5, np.inf), (2, 6, np.inf)], [(m - 1, 1056, np.nan)]):
            bad = clean.clone()
            for t, c, v in places:
                bad[t, c] = float(v)
            y = host(trmoe.moe_mx4(L, bad, k, score=score))
            hit = np.isin(np.arange(m), [t for t, _, _ in places])
            assert np.isnan(y[hit]).all() and np.array_equal(y[~hit], want[~hit])


@pytest.mark.parametrize("m,F", CHOICES)
def test_a_poisoned_token_that_chooses_nothing(m, F):
    """With the logits given and all masked: NaN where x is poisoned, zeros where it is not."""
    say(f"moe_mx4 poisoned, masked tokens m={m} F={F}")
    rng = np.random.default_rng(m + F)
    E, k, H = 12, 4, 100
    L, _, _, _, _ = layer_of(rng, E, H, F, router=False)
    x, logits = rng.standard_normal((m, H)).astype(np.float32), rng.standard_normal((m, E)).astype(np.float32)
    logits[:4] = -np.inf
    x[1, 99], x[3, 0], x[4, 40] = np.nan, -np.inf, np.nan
    y = host(trmoe.moe_mx4(L, dev(x), k, rlog=dev(logits)))
    nan = np.isin(np.arange(m), (1, 3, 4))
    assert np.isnan(y[nan]).all() and np.isfinite(y[~nan]).all()
    assert (y[[0, 2]] == 0).all() and (y[5:] != 0).any(1).all()


@pytest.mark.parametrize("xt", ["f32", "bf16"])
@pytest.mark.parametrize("m,F", CHOICES)
def test_values_near_the_largest(m, F, xt):
    """x up to the largest number, with weights so small that every sum is an ordinary one."""
    import torch
    say(f"moe_mx4 x near the largest m={m} F={F} {xt}")
    rng = np.random.default_rng(m + F)
    E, k, H = 6, 4, 200
    w = {"gate": rows4(rng, E, F, H, spread=2.0 ** -123), "up": rows4(rng, E, F, H, spread=2.0 ** -123),
         "down": rows4(rng, E, H, F, spread=0.1)}
    L = trmoe.MX4Layer(*[trmoe.MX4Weights(*apart(*w[i]), K) for i, K in (("gate", H), ("up", H), ("down", F))])
    x = (rng.uniform(2.9e38, 3.38e38, (m, H)) * rng.choice([-1, 0, 0, 0, 1], (m, H))).astype(np.float32)
    x[0, :32] = 3.38e38
    x[1, 64:96] = np.linspace(2.95e38, 3.01e38, 32)  # about the first part's border, 3.5 2^126
    xd = dev(x).to(i8ref.torch_dtype(xt))
    assert xd.isfinite().all()
    logits = (rng.permutation(m * E).reshape(m, E) / (m * E)).astype(np.float32)
    kw = dict(k=k, n_group=1, topk_group=1, group_top=2, renorm=True, factor=1.0)
    rid, rw, _ = i8ref.route(logits, bias=None, score="sigmoid", **kw)
    v = {i: R.values(*w[i], K) for i, K in (("gate", H), ("up", H), ("down", F))}
    want, tol = R.layer(host(xd).astype(np.float64), v["gate"], v["up"], v["down"], rid, rw, "f32")
    within(host(trmoe.moe_mx4(L, xd, rlog=dev(logits), score="sigmoid", dtype=torch.float32, **kw)), want, tol)


@pytest.mark.parametrize("m,F", CHOICES)
def test_activations_near_the_largest(m, F):
    """The same of h: silu(4) 2^126 is 3.34e38."""
    say(f"moe_mx4 h near the largest m={m} F={F}")
    rng = np.random.default_rng(m + F)
    E, k, H = 6, 4, 64
    one, flat = np.searchsorted(R.VALUES[:8], [1.0, 4.0]), {}
    for i, code, scale in (("gate", one[1], 127), ("up", one[0], 127 + 126)):
        c = np.zeros((E, F, H), np.uint8)
        c[:, :, 0] = code + (8 * rng.integers(0, 2, (E, F)) if i == "up" else 0)
        s = np.full((E, F, 2), 127, np.uint8)
        s[:, :, 0] = scale
        c[:, ::3, 0] = np.searchsorted(R.VALUES[:8], 1.0)  # every third row smaller by its gate or up
        if i == "up":
            c[:, ::3, 0] = np.searchsorted(R.VALUES[:8], 0.5)
        flat[i] = R.pack(c), s
    flat["down"] = rows4(rng, E, H, F, spread=2.0 ** -122)
    L = trmoe.MX4Layer(*[trmoe.MX4Weights(*apart(*flat[i]), K) for i, K in (("gate", H), ("up", H), ("down", F))])
    x = np.zeros((m, H), np.float32)
    x[:, 0], x[:, 40] = 1.0, np.arange(m)  # the second value meets zeros
    logits = (rng.permutation(m * E).reshape(m, E) / (m * E)).astype(np.float32)
    kw = dict(k=k, n_group=1, topk_group=1, group_top=2, renorm=True, factor=1.0)
    rid, rw, _ = i8ref.route(logits, bias=None, score="sigmoid", **kw)
    v = {i: R.values(*flat[i], K) for i, K in (("gate", H), ("up", H), ("down", F))}
    h = R.silu(v["gate"][0, :, 0]) * v["up"][0, :, 0]
    assert 3.3e38 < np.abs(h).max() < 3.4e38
    want, tol = R.layer(x.astype(np.float64), v["gate"], v["up"], v["down"], rid, rw, "f32")
    within(host(trmoe.moe_mx4(L, dev(x), rlog=dev(logits), score="sigmoid", **kw)), want, tol)


# ---- the choice in 64 bits ---------------------------------------------------------------------------

def alike(rng, m, E, kind):
    """Logits that 32 bits do not decide: all alike, alike but for a few, in runs of a hundred."""
    l = np.full((m, E), 0.25, np.float32)
    if kind == "few":
        l[:, ::37] = 0.5
        l[m - 1, 5] = -np.inf
    if kind == "runs":
        l = (np.arange(E) // 100)[None, :].repeat(m, 0).astype(np.float32) / 8
    return l


@pytest.mark.parametrize("E,k,score,bias,groups,keep,renorm", [
    (300, 5, "sigmoid", False, 1, 1, True), (300, 5, "softmax", False, 1, 1, False), (300, 32, "softmax", True, 1, 1, True),
    (1024, 7, "sigmoid", True, 4, 2, True), (1024, 4, "softmax", False, 2, 1, True), (256, 8, "sigmoid", True, 8, 4, False)])
@pytest.mark.parametrize("kind", ["all", "few", "runs"])
@pytest.mark.parametrize("m,F", [(2, 40), (8, 1100)])
def test_a_choice_among_equals(m, F, kind, E, k, score, bias, groups, keep, renorm):
    """More than 64 candidates: every key in 64 bits, the lower index first.  By route_scores' choice of the same logits."""
    import torch
    say(f"moe_mx4 equal logits m={m} F={F} {kind} E={E} k={k} {score} bias={bias} groups={groups}")
    rng = np.random.default_rng(E + k)
    H = 32
    if F > 100 and E > 256:
        E //= 4  # fewer experts where they are wide: 75 and more stay in question
    L, w, _, b, _ = layer_of(rng, E, H, F, bias=bias, router=False)
    if bias:
        L.bias.fill_(0.125)
    x = rng.standard_normal((m, H)).astype(np.float32)
    logits = alike(rng, m, E, kind)
    kw = dict(score=score, n_group=groups, topk_group=keep, renorm=renorm, factor=1.5)
    ids, wt, n = trmoe.route_scores(dev(logits), k, bias=L.bias, **kw)
    want_ids, _, want_n = i8ref.route(logits, k, None if b is None else np.full(E, 0.125), score, groups, keep, 2, renorm, 1.5)
    assert np.array_equal(host(n), want_n) and np.array_equal(host(ids)[:, :k], want_ids)
    y = host(trmoe.moe_mx4(L, dev(x), k, rlog=dev(logits), **kw))
    want, tol = R.layer(x.astype(np.float64), w["gate"], w["up"], w["down"], host(ids)[:, :k], host(wt)[:, :k].astype(np.float64), "f32")
    within(y, want, tol)
    assert torch.equal(trmoe.moe_mx4(L, dev(x), k, rlog=dev(logits), **kw), dev(y))


@pytest.mark.parametrize("m,F", CHOICES)
def test_a_logit_of_infinity(m, F):
    """Under softmax it makes the row's scores NaN: chosen by the logits without a bias, with NaN weights; with one nothing is
    chosen.  Under sigmoid it is the largest."""
    say(f"moe_mx4 infinite logits m={m} F={F}")
    rng = np.random.default_rng(m + F)
    E, k, H = 20, 4, 96
    x, logits = rng.standard_normal((m, H)).astype(np.float32), rng.standard_normal((m, E)).astype(np.float32)
    logits[2, 7] = np.inf
    for bias in (False, True):
        L, w, _, b, _ = layer_of(rng, E, H, F, bias=bias, router=False)
        for score in ("softmax", "sigmoid"):
            ids, wt, n = trmoe.route_scores(dev(logits), k, bias=L.bias, score=score)
            y = host(trmoe.moe_mx4(L, dev(x), k, rlog=dev(logits), score=score))
            ids, wt, n = host(ids)[:, :k], host(wt)[:, :k].astype(np.float64), host(n)
            rows = np.arange(m)
            if score == "softmax":
                assert n[2] == (0 if bias else k)
                assert (y[2] == 0).all() if bias else np.isnan(y[2]).all()
                rows = np.delete(rows, 2)
            want, tol = R.layer(x[rows].astype(np.float64), w["gate"], w["up"], w["down"], ids[rows], wt[rows], "f32")
            within(y[rows], want, tol)
