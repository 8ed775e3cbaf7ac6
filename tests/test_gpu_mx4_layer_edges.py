"""The layer on 4-bit experts where its activations are no numbers."""
from __future__ import annotations

import i8ref
import numpy as np
import pytest

import trmoe
from test_gpu_mx4 import dev, host, layer_of, say

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
