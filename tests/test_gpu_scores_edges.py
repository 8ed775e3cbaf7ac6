"""Routing by scores at the ends of its types, on the GPU against the plain 64-bit form (tests/i8ref.py)."""
from __future__ import annotations

import i8ref as R
import numpy as np
import pytest

import trmoe
from test_gpu_scores_i8 import dev, host, say

pytestmark = pytest.mark.gpu
LOW = np.finfo(np.float32).min


def check_route(lg, bias, score, rtol=2.0 ** -22, **kw):
    """ids and n_sel equal, weights within rtol."""
    kw = {**dict(n_group=1, topk_group=1, group_top=2, renorm=True, factor=1.0), **kw}
    ids, w, n = trmoe.route_scores(dev(lg), bias=None if bias is None else dev(bias), score=score, **kw)
    rid, rw, rn = R.route(lg, bias=bias, score=score, **kw)
    assert np.array_equal(host(n), rn), (host(n), rn)
    assert np.array_equal(host(ids)[:, :kw["k"]], rid)
    np.testing.assert_allclose(host(w)[:, :kw["k"]], rw, rtol=rtol, atol=2.0 ** -149)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,groups,keep,k", [(16, 4, 2, 8), (256, 8, 4, 32), (256, 8, 8, 8), (1020, 17, 3, 32), (12, 6, 5, 9)])
@pytest.mark.parametrize("low", [LOW, -2e38, "spread"])
def test_groups_whose_sums_leave_the_type(score, E, groups, keep, k, low):
    """Two keys of a group near the lowest number: their sum is below it, and the group is there all the same."""
    say(f"route_scores group sums out of range {score} E={E} {groups}/{keep} {low}")
    rng = np.random.default_rng(E + k)
    lg = rng.standard_normal((12, E)).astype(np.float32)
    gs = E // groups
    bias = np.full(E, LOW, np.float32)
    bias[:] = rng.choice(np.array([LOW, -3e38, -2.5e38, -1.8e38], np.float32), E) if low == "spread" else low
    bias[:gs] = 0.0                       # one group as usual
    lg[1, :gs] = -np.inf                  # and none
    lg[2, gs:2 * gs] = -np.inf            # a group with nothing to choose
    lg[3, 2 * gs + 1:3 * gs] = -np.inf    # with one
    lg[4, gs:] = -np.inf
    for top in (1, 2):
        check_route(lg, bias, score, k=k, n_group=groups, topk_group=keep, group_top=top)
    high = -bias
    check_route(lg, high, score, k=k, n_group=groups, topk_group=keep)


@pytest.mark.parametrize("E,k,groups,keep,bias", [(5, 5, 1, 1, False), (256, 8, 1, 1, False), (512, 10, 1, 1, True),
                                                  (1024, 32, 32, 5, True), (160, 6, 8, 3, False)])
def test_softmax_weights_left_as_they_are(E, k, groups, keep, bias):
    """Not renormalised, a weight is exp(l - max) / sum in 64 bits, rounded once."""
    say(f"route_scores softmax weights E={E} k={k} {groups}/{keep} bias={bias}")
    rng = np.random.default_rng(E + k)
    lg = (rng.standard_normal((400, E)) * rng.uniform(0.1, 6.0, (400, 1))).astype(np.float32)
    lg[rng.random(lg.shape) < 0.05] = -np.inf
    lg[7] = lg[7, 0] if np.isfinite(lg[7, 0]) else 0.25  # all alike
    b = (rng.standard_normal(E) * 0.1).astype(np.float32) if bias else None
    if bias:
        b[::9] = -np.inf  # not to be chosen, but part of the sum
    # half a step, and what 64-bit exponentials and their sum may differ by
    check_route(lg, b, "softmax", rtol=1.001 * R.EPS["f32"], k=k, n_group=groups, topk_group=keep, renorm=False)


def test_an_infinite_logit():
    """A softmax row with a logit of +inf has NaN scores: nothing is chosen where they enter the choice, else NaN weights.  Its
    sigmoid is 1."""
    say("route_scores infinite logits")
    E, k = 16, 3
    lg = np.random.default_rng(4).standard_normal((3, E)).astype(np.float32)
    lg[1, 9] = np.inf
    lg[2, [2, 9]] = np.inf
    bias = np.zeros(E, np.float32)
    base = dict(k=k, n_group=1, topk_group=1, group_top=2, renorm=True, factor=1.0)
    for kw, b, scored in ((base, None, False), (base, bias, True), ({**base, "n_group": 4, "topk_group": 2}, None, True),
                          ({**base, "n_group": 4, "topk_group": 2, "group_top": 1}, None, False)):
        ids, w, n = (host(t) for t in trmoe.route_scores(dev(lg), bias=None if b is None else dev(b), score="softmax", **kw))
        assert n[0] == k and np.isfinite(w[0, :k]).all()
        if scored:
            assert (n[1:] == 0).all() and (ids[1:, :k] == -1).all() and (w[1:, :k] == 0).all()
        else:
            assert (n[1:] == k).all() and ids[1, 0] == 9 and ids[2, :2].tolist() == [2, 9] and np.isnan(w[1:, :k]).all()
        check_route(lg, b, "sigmoid", **kw)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("bias", [False, True])
def test_choices_that_hang_on_no_rounding(score, bias):
    """Every logit moved by up to 1e-12 of itself, each by another amount: the plain form's choice stays, so the kernel's has to be
    the same."""
    say(f"route_scores settled {score} bias={bias}")
    rng = np.random.default_rng(17 + bias)
    lg = (rng.standard_normal((200, 256)) * 1.5).astype(np.float32)
    lg[rng.random(lg.shape) < 0.05] = -np.inf
    b = (rng.standard_normal(256) * 0.1).astype(np.float32) if bias else None
    kw = dict(k=8, n_group=8, topk_group=4, group_top=2, renorm=True, factor=2.5)
    moved = np.where(np.isfinite(lg), lg.astype(np.float64) * (1 + rng.uniform(-1e-12, 1e-12, lg.shape)), lg)
    assert np.array_equal(R.route(lg, bias=b, score=score, **kw)[0], R.route(moved, bias=b, score=score, **kw)[0])
    check_route(lg, b, score, **kw)
