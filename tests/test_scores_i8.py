"""Refusals of routing by scores and the int8 products, at the C entry points and in the Python calls, without a GPU:
a bad argument is a status with a message and no device work."""
from __future__ import annotations

import ctypes as C

import pytest

import trmoe

P = C.c_void_p(256)  # 16-byte aligned, never touched


def err():
    return trmoe.lib().trk_last_error().decode()


def policy(**kw):
    d = dict(k=8, score=1, n_group=1, topk_group=1, group_top=2, renorm=1, factor=1.0)
    d.update(kw)
    return trmoe.ScorePolicy(*[d[f] for f, _ in trmoe.ScorePolicy._fields_])


def mat(**kw):
    d = dict(ptr=256, scale=256, rows=64, k=100, count=4, ld=112, stride=112 * 64)
    d.update(kw)
    return trmoe.I8Mat(*[d[f] for f, _ in trmoe.I8Mat._fields_])


@pytest.mark.parametrize("kw,E,rc,word", [
    (dict(k=0), 64, -2, "k (0)"), (dict(k=33), 64, -2, "k (33)"), (dict(k=9), 8, -2, "k (9)"),
    (dict(score=2), 64, -2, "score"), (dict(n_group=0), 64, -2, "n_group"), (dict(n_group=3), 64, -2, "n_group"),
    (dict(n_group=64), 64, -2, "n_group"), (dict(n_group=4, topk_group=5), 64, -2, "topk_group"),
    (dict(n_group=4, topk_group=0), 64, -2, "topk_group"), (dict(group_top=3), 64, -2, "group_top"),
    (dict(factor=float("inf")), 64, -2, "factor"), (dict(factor=float("nan")), 64, -2, "factor"),
    ({}, 0, -1, "n_expert"), ({}, 1025, -1, "n_expert")])
def test_route_scores_refuses(kw, E, rc, word):
    p = policy(**kw)
    assert trmoe.lib().trk_route_scores(P, None, 1, E, C.byref(p), P, P, P, None) == rc and word in err()


def test_route_scores_null_and_nothing_to_do():
    L, p = trmoe.lib(), policy()
    assert L.trk_route_scores(P, None, 1, 64, None, P, P, P, None) == -1
    assert L.trk_route_scores(None, None, 1, 64, C.byref(p), P, P, P, None) == -1 and "null" in err()
    assert L.trk_route_scores(None, None, 0, 64, C.byref(p), None, None, None, None) == 0


@pytest.mark.parametrize("args,word", [
    ((P, 3, 64, 2, 64, P, 64, P), "element type"), ((P, 0, 64, 2, 0, P, 64, P), "k must"),
    ((P, 0, 63, 2, 64, P, 64, P), "stride"), ((P, 0, 64, 2, 64, P, 63, P), "stride"),
    ((C.c_void_p(258), 0, 64, 2, 64, P, 64, P), "aligned"), ((C.c_void_p(257), 1, 64, 2, 64, P, 64, P), "aligned"),
    ((None, 0, 64, 2, 64, P, 64, P), "null")])
def test_quantize_rows_refuses(args, word):
    assert trmoe.lib().trk_quantize_rows(*args, None) == -1 and word in err()


def gemm(w=None, item=0, q=P, ldq=112, scale=P, m=3, bias=None, y=P, dtype=0, ldy=64, acc=0):
    return trmoe.lib().trk_gemm_i8(C.byref(w or mat()), item, q, ldq, scale, m, bias, y, dtype, ldy, acc, None)


@pytest.mark.parametrize("kw,word", [
    (dict(w=mat(ptr=264)), "multiples of 16"), (dict(w=mat(ld=104)), "multiples of 16"), (dict(w=mat(ld=96)), "below k"),
    (dict(w=mat(k=131072, ld=131072)), "above 131071"), (dict(w=mat(stride=112 * 64 - 16)), "stride"),
    (dict(w=mat(stride=112 * 64 + 8)), "stride"), (dict(w=mat(rows=0)), "empty"), (dict(w=mat(k=0)), "empty"),
    (dict(w=mat(count=0)), "empty"), (dict(w=mat(scale=0)), "null"), (dict(item=4), "item"), (dict(q=C.c_void_p(260)), "q:"),
    (dict(ldq=100), "q:"), (dict(ldq=96), "below k"), (dict(dtype=3), "element type"), (dict(y=C.c_void_p(258)), "aligned"),
    (dict(ldy=63), "ldy"), (dict(q=None), "null"), (dict(y=None), "null")])
def test_gemm_i8_refuses(kw, word):
    assert gemm(**kw) == -1 and word in err()


def test_gemm_i8_nothing_to_do():
    assert gemm(m=0, q=None, scale=None, y=None) == 0


def words(m, slots, E):
    n = C.c_uint64()
    assert trmoe.lib().trk_experts_plan_words(m, slots, E, C.byref(n)) == 0
    return n.value


def test_experts_entry_counts_are_checked():
    L, n = trmoe.lib(), C.c_uint64()
    for m, slots, E, word in [(1, 0, 8, "slots"), (1, 33, 8, "slots"), (1, 1, 0, "n_expert"), (1, 1, 1025, "n_expert"),
                              (1 << 27, 16, 8, "too large")]:
        assert L.trk_experts_plan_words(m, slots, E, C.byref(n)) == -1 and word in err()
        assert L.trk_experts_plan(P, P, m, slots, E, P, None) == -1 and word in err()
        assert L.trk_experts_down_work_bytes(m, slots, E, 64, C.byref(n)) == -1 and word in err()
    assert L.trk_experts_plan_words(1, 1, 8, None) == -1
    assert words(0, 4, 8) == 0 and words(1, 8, 256) == 0  # one token takes no plan
    assert words(4096, 10, 512) >= 4 + 40960
    assert words(trmoe.EXPERTS_DIRECT_M, 10, 512) == 0 and words(trmoe.EXPERTS_DIRECT_M + 1, 10, 512) > 0


def up(gate=None, up_=None, q=P, ldq=112, m=4096, ids=P, slots=2, plan=P, h=P, dtype=0, ldh=64):
    return trmoe.lib().trk_experts_up_i8(C.byref(gate or mat()), C.byref(up_ or mat()), q, ldq, P, m, ids, P, slots, plan,
                                         h, dtype, ldh, None)


@pytest.mark.parametrize("kw,word", [
    (dict(up_=mat(rows=63)), "differ"), (dict(up_=mat(k=99)), "differ"), (dict(up_=mat(count=3)), "differ"),
    (dict(gate=mat(ptr=8)), "multiples"), (dict(up_=mat(ptr=8)), "multiples"), (dict(slots=0), "slots"),
    (dict(ldh=63), "ldh"), (dict(plan=None), "plan"), (dict(plan=C.c_void_p(264)), "plan"), (dict(ids=None), "null"),
    (dict(h=C.c_void_p(255)), "aligned"), (dict(dtype=7), "element type"), (dict(ldq=16), "below k")])
def test_experts_up_refuses(kw, word):
    assert up(**kw) == -1 and word in err()


def down(w=None, q=P, ldq=112, m=4096, ids=P, wt=P, slots=2, plan=P, work=P, y=P, dtype=0, ldy=64):
    return trmoe.lib().trk_experts_down_i8(C.byref(w or mat()), q, ldq, P, m, ids, wt, P, slots, plan, work, y, dtype, ldy,
                                           0, None)


@pytest.mark.parametrize("kw,word", [
    (dict(w=mat(count=1025)), "n_expert"), (dict(slots=40), "slots"), (dict(ldy=63), "ldy"), (dict(plan=None), "plan"),
    (dict(work=None), "work"), (dict(work=C.c_void_p(260)), "work"), (dict(wt=None), "null"),
    (dict(y=C.c_void_p(255)), "aligned"), (dict(ldq=104), "multiples")])
def test_experts_down_refuses(kw, word):
    assert down(**kw) == -1 and word in err()


def test_experts_nothing_to_do():
    assert up(m=0, q=None, ids=None, plan=None, h=None) == 0
    assert down(m=0, q=None, ids=None, wt=None, plan=None, work=None, y=None) == 0


def test_python_calls_refuse_tensors_elsewhere_and_of_wrong_shape():
    import torch
    q, s = torch.zeros((3, 32), dtype=torch.int8), torch.ones(3)
    with pytest.raises(trmoe.TrkError, match="on the GPU"):
        trmoe.quantize_rows(torch.zeros((3, 32)))
    with pytest.raises(trmoe.TrkError, match="contiguous"):
        trmoe.quantize_rows(torch.zeros((32, 3)).t())
    with pytest.raises(trmoe.TrkError, match="on the GPU"):
        trmoe.I8Weights(q, s)
    with pytest.raises(trmoe.TrkError, match="weight scales"):
        trmoe.I8Weights(q, torch.ones(4))
    with pytest.raises(trmoe.TrkError, match="int8"):
        trmoe.I8Weights(q.float(), s)
    with pytest.raises(trmoe.TrkError, match="storage ends"):
        trmoe._whole_pieces(torch.zeros(33, dtype=torch.int8)[1:], 2, 16, 16 + 1, "q")
    with pytest.raises(trmoe.TrkError, match="logits"):
        trmoe.route_scores(torch.zeros((2, 8), dtype=torch.float64), 2)
    with pytest.raises(trmoe.TrkError, match="score"):
        trmoe.route_scores(torch.zeros((2, 8)), 2, score="max")
    with pytest.raises(trmoe.TrkError, match="bias"):
        trmoe.route_scores(torch.zeros((2, 8)), 2, bias=torch.zeros(7))
    with pytest.raises(trmoe.TrkError, match="ids"):
        trmoe.experts_plan(torch.zeros((2, 8), dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 2, 8)


def test_forms_and_plan_extents_on_the_host(tmp_path):
    """The rules that choose a form, at sizes where the forms were timed, and the plan's sizes under any load."""
    import os
    import subprocess
    here = os.path.dirname(os.path.abspath(__file__))
    exe = str(tmp_path / "i8_rules_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", os.path.join(here, "i8_rules_check.cpp"), "-o", exe],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.startswith("ok"), r.stdout
