"""Refusals of the microscaled 4-bit calls, at the C entry points and in the Python calls, without a GPU: a bad argument is a
status with a message and no device work."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import mx4ref as R
import trmoe

P = C.c_void_p(256)  # 16-byte aligned, never touched


def err():
    return trmoe.lib().trk_last_error().decode()


def mat(**kw):  # k = 100: four blocks
    d = dict(ptr=256, scale=256, rows=64, k=100, count=4, ld=64, stride=64 * 64, scale_ld=4, scale_stride=4 * 64)
    d.update(kw)
    return trmoe.Mx4Mat(*[d[f] for f, _ in trmoe.Mx4Mat._fields_])


def policy(**kw):
    d = dict(k=2, score=1, n_group=1, topk_group=1, group_top=2, renorm=1, factor=1.0)
    d.update(kw)
    return trmoe.ScorePolicy(*[d[f] for f, _ in trmoe.ScorePolicy._fields_])


MATS = [(dict(ptr=264), "multiples of 16"), (dict(ld=72), "multiples of 16"), (dict(ld=48), "below 64 bytes"),
        (dict(scale=258), "multiples of 4"), (dict(scale_ld=6), "multiples of 4"), (dict(scale_ld=0), "below 4 blocks"),
        (dict(k=(1 << 30) + 1, ld=1 << 34), "k ("), (dict(stride=64 * 64 - 16), "stride"), (dict(stride=64 * 64 + 8), "stride"),
        (dict(scale_stride=4 * 64 - 4), "scales' stride"), (dict(scale_stride=4 * 64 + 2), "scales' stride"),
        (dict(rows=0), "empty"), (dict(k=0), "empty"), (dict(count=0), "empty"), (dict(scale=0), "null"), (dict(ptr=0), "null"),
        (dict(rows=0xffffff01, count=1), "rows"), (dict(ld=1 << 41, count=1), "too large")]


@pytest.mark.parametrize("args,word", [
    ((P, 3, 64, 2, 64, P, 32, P, 4), "element type"), ((P, 0, 64, 2, 0, P, 32, P, 4), "k (0)"),
    ((P, 0, 63, 2, 64, P, 32, P, 4), "below k"), ((P, 0, 64, 2, 64, P, 16, P, 4), "below 32 bytes"),
    ((P, 0, 64, 2, 64, P, 40, P, 4), "multiples of 16"), ((P, 0, 64, 2, 64, C.c_void_p(264), 32, P, 4), "multiples of 16"),
    ((P, 0, 64, 2, 64, P, 32, P, 2), "multiples of 4"), ((P, 0, 64, 2, 64, P, 32, P, 0), "below 2 blocks"),
    ((P, 0, 64, 2, 64, P, 32, C.c_void_p(258), 4), "multiples of 4"), ((C.c_void_p(258), 0, 64, 2, 64, P, 32, P, 4), "aligned"),
    ((C.c_void_p(257), 1, 64, 2, 64, P, 32, P, 4), "aligned"), ((None, 0, 64, 2, 64, P, 32, P, 4), "null"),
    ((P, 0, 64, 2, (1 << 30) + 1, P, 32, P, 4), "k (")])
def test_quantize_refuses(args, word):
    assert trmoe.lib().trk_quantize_mx4(*args, None) == -1 and word in err()


@pytest.mark.parametrize("args,word", [
    ((P, 32, P, 4, 2, 64, P, 3, 64), "element type"), ((P, 32, P, 4, 2, 0, P, 0, 64), "k (0)"),
    ((P, 32, P, 4, 2, 64, P, 0, 63), "below k"), ((P, 16, P, 4, 2, 64, P, 0, 64), "below 32 bytes"),
    ((P, 32, P, 3, 2, 64, P, 0, 64), "multiples of 4"), ((P, 32, P, 4, 2, 64, C.c_void_p(258), 0, 64), "aligned"),
    ((None, 32, P, 4, 2, 64, P, 0, 64), "null"), ((P, 32, None, 4, 2, 64, P, 0, 64), "null"), ((P, 32, P, 4, 2, 64, None, 0, 64), "null")])
def test_dequantize_refuses(args, word):
    assert trmoe.lib().trk_dequantize_mx4(*args, None) == -1 and word in err()


def gemm(w=None, item=0, q=P, ldq=64, scale=P, lds=4, m=3, bias=None, y=P, dtype=0, ldy=64, acc=0):
    return trmoe.lib().trk_gemm_mx4(C.byref(w or mat()), item, q, ldq, scale, lds, m, bias, y, dtype, ldy, acc, None)


@pytest.mark.parametrize("kw,word", [(dict(w=mat(**kw)), word) for kw, word in MATS] + [
    (dict(item=4), "item"), (dict(q=C.c_void_p(260)), "q:"), (dict(ldq=72), "q:"), (dict(ldq=48), "below 64"), (dict(lds=2), "q:"),
    (dict(lds=0), "below 4"), (dict(dtype=3), "element type"), (dict(y=C.c_void_p(258)), "aligned"), (dict(ldy=63), "ldy"),
    (dict(q=None), "null"), (dict(scale=None), "null"), (dict(y=None), "null"), (dict(m=0xffffff01), "m (")])
def test_gemm_refuses(kw, word):
    assert gemm(**kw) == -1 and word in err()


def up(gate=None, up_=None, q=P, ldq=64, lds=4, m=4096, ids=P, slots=2, plan=P, h=P, dtype=0, ldh=64):
    return trmoe.lib().trk_experts_up_mx4(C.byref(gate or mat()), C.byref(up_ or mat()), q, ldq, P, lds, m, ids, P, slots, plan,
                                          h, dtype, ldh, None)


@pytest.mark.parametrize("kw,word", [
    (dict(up_=mat(rows=63)), "differ"), (dict(up_=mat(k=99)), "differ"), (dict(up_=mat(count=3)), "differ"),
    (dict(gate=mat(ptr=8)), "multiples"), (dict(up_=mat(ptr=8)), "multiples"), (dict(slots=0), "slots"), (dict(slots=33), "slots"),
    (dict(ldh=63), "ldh"), (dict(plan=None), "plan"), (dict(plan=C.c_void_p(264)), "plan"), (dict(ids=None), "null"),
    (dict(h=C.c_void_p(255)), "aligned"), (dict(dtype=7), "element type"), (dict(ldq=16), "below 64"), (dict(lds=0), "below 4")])
def test_experts_up_refuses(kw, word):
    assert up(**kw) == -1 and word in err()


def down(w=None, q=P, ldq=64, lds=4, m=4096, ids=P, wt=P, slots=2, plan=P, work=P, y=P, dtype=0, ldy=64):
    return trmoe.lib().trk_experts_down_mx4(C.byref(w or mat()), q, ldq, P, lds, m, ids, wt, P, slots, plan, work, y, dtype,
                                            ldy, 0, None)


@pytest.mark.parametrize("kw,word", [
    (dict(w=mat(count=1025)), "n_expert"), (dict(slots=40), "slots"), (dict(ldy=63), "ldy"), (dict(plan=None), "plan"),
    (dict(work=None), "work"), (dict(work=C.c_void_p(260)), "work"), (dict(wt=None), "null"),
    (dict(y=C.c_void_p(255)), "aligned"), (dict(ldq=56), "multiples")])
def test_experts_down_refuses(kw, word):
    assert down(**kw) == -1 and word in err()


def layer_w(router=256, bias=0, shared_gate=0, gate=None, up=None, down=None, n_shared=0):
    back = mat(rows=100, k=64, ld=32, stride=32 * 100, scale_ld=4, scale_stride=400)
    return trmoe.MoeMx4W(router, bias, shared_gate, gate or mat(), up or mat(), down or back, n_shared)


def moe(w=None, p=None, x=P, xdt=0, ldx=100, rlog=None, m=3, work=P, y=P, ydt=0, ldy=100):
    return trmoe.lib().trk_moe_mx4(C.byref(w or layer_w()), C.byref(p or policy()), x, xdt, ldx, rlog, m, work, y, ydt, ldy, None)


@pytest.mark.parametrize("kw,rc,word", [
    (dict(w=layer_w(up=mat(rows=63))), -1, "differ"), (dict(w=layer_w(down=mat())), -1, "go back"),
    (dict(w=layer_w(gate=mat(ptr=8))), -1, "multiples"), (dict(w=layer_w(n_shared=4)), -1, "n_expert"),
    (dict(w=layer_w(n_shared=33)), -1, "n_shared"),
    (dict(w=layer_w(gate=mat(rows=(1 << 24) + 1, count=1), up=mat(rows=(1 << 24) + 1, count=1),
                    down=mat(rows=100, k=(1 << 24) + 1, ld=1 << 23 | 16, scale_ld=1 << 20, count=1)), p=policy(k=1)), -1, "at most"), (dict(w=layer_w(router=0)), -1, "router"), (dict(m=9), -3, "m (9)"),
    (dict(p=policy(k=5)), -2, "k (5)"), (dict(p=policy(k=0)), -2, "k (0)"), (dict(w=layer_w(n_shared=3)), -2, "k (2)"),
    (dict(p=policy(n_group=3)), -2, "n_group"), (dict(p=policy(factor=float("nan"))), -2, "factor"),
    (dict(xdt=3), -1, "element type"), (dict(ydt=3), -1, "element type"), (dict(ldx=99), -1, "stride"), (dict(ldy=99), -1, "stride"),
    (dict(x=None), -1, "null"), (dict(y=None), -1, "null"), (dict(work=None), -1, "null"), (dict(work=C.c_void_p(260)), -1, "work"),
    (dict(x=C.c_void_p(258)), -1, "aligned"), (dict(y=C.c_void_p(258)), -1, "aligned")])
def test_layer_refuses(kw, rc, word):
    assert moe(**kw) == rc and word in err()


def test_layer_work():
    L, n, w = trmoe.lib(), C.c_uint64(), layer_w(n_shared=1)
    assert L.trk_moe_mx4_work_bytes(C.byref(w), 2, 3, None) == -1
    assert L.trk_moe_mx4_work_bytes(C.byref(w), 2, 9, C.byref(n)) == -3
    assert L.trk_moe_mx4_work_bytes(C.byref(w), 4, 3, C.byref(n)) == -2  # three routed experts
    assert L.trk_moe_mx4_work_bytes(C.byref(w), 2, 3, C.byref(n)) == 0
    assert n.value >= 4 * (3 * 3 + 3 + 2 * 3 * 32 + 3 + 3 * 3 * 64) and n.value % 16 == 0
    assert L.trk_moe_mx4_work_bytes(C.byref(w), 2, 0, C.byref(n)) == 0 and n.value == 0


def test_nothing_to_do():
    L = trmoe.lib()
    assert L.trk_quantize_mx4(None, 0, 64, 0, 64, None, 32, None, 4, None) == 0
    assert L.trk_dequantize_mx4(None, 32, None, 4, 0, 64, None, 0, 64, None) == 0
    assert gemm(m=0, q=None, scale=None, y=None) == 0
    assert up(m=0, q=None, ids=None, plan=None, h=None) == 0
    assert down(m=0, q=None, ids=None, wt=None, plan=None, work=None, y=None) == 0
    assert moe(m=0, x=None, work=None, y=None) == 0


def test_python_calls_refuse():
    import torch
    q, s = torch.zeros((3, 32), dtype=torch.uint8), torch.zeros((3, 4), dtype=torch.uint8)
    with pytest.raises(trmoe.TrkError, match="on the GPU"):
        trmoe.quantize_mx4(torch.zeros((3, 32)))
    with pytest.raises(trmoe.TrkError, match="contiguous"):
        trmoe.quantize_mx4(torch.zeros((32, 3)).t())
    with pytest.raises(trmoe.TrkError, match="on the GPU"):
        trmoe.MX4Weights(q, s[:, :2], 64)
    with pytest.raises(trmoe.TrkError, match="k = 65"):
        trmoe.MX4Weights(q, s[:, :2], 65)
    with pytest.raises(trmoe.TrkError, match="k = 0"):
        trmoe.MX4Weights(q[:, :0], s[:, :0], 0)
    with pytest.raises(trmoe.TrkError, match="uint8"):
        trmoe.MX4Weights(q.float(), s, 64)
    with pytest.raises(trmoe.TrkError, match="k = 32"):
        trmoe.dequantize_mx4(q, s[:, :2], 32)
    with pytest.raises(trmoe.TrkError, match="contiguous"):
        trmoe.dequantize_mx4(q, s.as_strided((3, 2), (4, 2)), 64)
    with pytest.raises(trmoe.TrkError, match="storage ends"):
        trmoe.dequantize_mx4(q, torch.zeros((3, 2), dtype=torch.uint8), 64)
    with pytest.raises(trmoe.TrkError, match="32 bits"):
        trmoe.dequantize_mx4(q, s, 1 << 32)


def test_forms_on_the_host(tmp_path):
    """The rules that choose a form, at sizes where the forms were timed."""
    import os
    import subprocess
    here = os.path.dirname(os.path.abspath(__file__))
    exe = str(tmp_path / "mx4_rules_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", os.path.join(here, "mx4_rules_check.cpp"), "-o", exe],
                   check=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    assert out.startswith("ok"), out


def test_the_plain_form_rounds_as_it_says():
    x = np.zeros((1, 32), np.float32)
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9]
    x[0, :8], x[0, 8:16] = ties, -np.array(ties)
    c, s = R.quantize(x)
    assert s[0, 0] == 127 and R.VALUES[c[0, :8]].tolist() == [0, 1, 1, 2, 2, 4, 4, 6]
    assert c[0, 8:16].tolist() == [8 + v for v in c[0, :8]]
    assert R.quantize(x[:, 16:])[1][0, 0] == 0
