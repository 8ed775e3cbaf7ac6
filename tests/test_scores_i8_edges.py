"""Routing by scores and the int8 products without a GPU: what their calls do at the ends of their arguments."""
from __future__ import annotations

import contextlib

import pytest

import trmoe


def test_weights_are_laid_out_on_the_stream_given(monkeypatch):
    """quantize_weights copies weights whose rows are no one matrix; the copy belongs to the stream that reads it."""
    import torch
    on, st = [], object()

    @contextlib.contextmanager
    def stream(s):
        on.append(s)
        yield
        on.pop()

    class Sliced:
        """[4][6][32] rows of a wider stack"""
        shape = (4, 6, 32)

        def dim(self):
            return 3

        def reshape(self, *shape):
            assert shape == (-1, 32)
            return list(on)  # the streams entered where the copy is queued

    class Reached(Exception):
        pass

    def quantize_rows(flat, stream=None):
        raise Reached(flat, stream)

    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(trmoe, "quantize_rows", quantize_rows)
    for given in (st, None):
        with pytest.raises(Reached) as e:
            trmoe.quantize_weights(Sliced(), stream=given)
        assert e.value.args == ([st] if given else [], given)
    assert not on


def test_sizes_past_32_bits_are_refused():
    """The C entry points take 32-bit sizes: a longer tensor would be cut to its size modulo 2^32."""
    import torch

    def meta(*shape, dtype=torch.int8):
        return torch.empty(shape, dtype=dtype, device="meta")

    far = (1 << 32) + 64
    with pytest.raises(trmoe.TrkError, match="32 bits"):
        trmoe.quantize_rows(meta(1, far, dtype=torch.bfloat16))
    with pytest.raises(trmoe.TrkError, match="32 bits"):
        trmoe.quantize_rows(meta(far, 16, dtype=torch.bfloat16))
    for shape in ((1, far), (far, 16), (far, 2, 16)):
        with pytest.raises(trmoe.TrkError, match="32 bits"):
            trmoe.I8Weights(meta(*shape), meta(*shape[:-1], dtype=torch.float32))
    with pytest.raises(trmoe.TrkError, match="32 bits"):
        trmoe.route_scores(meta(far, 8, dtype=torch.float32), 2)

    class W:  # a matrix [5][64]: only its sizes are looked at before the rows'
        rows, k, count = 5, 64, 1
    with pytest.raises(trmoe.TrkError, match="32 bits"):
        trmoe.gemm_i8(W, meta(far, 64), meta(far, dtype=torch.float32))


def test_numbers_past_32_bits_are_refused():
    import torch
    far = (1 << 32) + 2
    lg = torch.zeros((2, 8))
    for kw in (dict(k=far), dict(k=2, n_group=far), dict(k=2, topk_group=far - 1), dict(k=2, group_top=far), dict(k=-1)):
        with pytest.raises(trmoe.TrkError, match="32 bits"):
            trmoe.route_scores(lg, **kw)
    ids, n = torch.zeros((9, 32), dtype=torch.int32), torch.zeros(9, dtype=torch.int32)
    with pytest.raises(trmoe.TrkError, match="32 bits"):
        trmoe.experts_plan(ids, n, far, 8)
    with pytest.raises(trmoe.TrkError, match="32 bits"):
        trmoe.experts_plan(ids, n, 2, far)
    class W:
        rows, k, count = 5, 64, 1
    q, s = torch.zeros((2, 64), dtype=torch.int8), torch.ones(2)
    for slots in (far, -1):
        with pytest.raises(trmoe.TrkError, match="32 bits"):
            trmoe.experts_up_i8(W, W, q, s, ids[:2], n[:2], slots)
    for item in (1, far - 2, -1):
        with pytest.raises(trmoe.TrkError, match="item"):
            trmoe.gemm_i8(W, q, s, item=item)


def test_rows_that_a_tile_cannot_number_are_refused():
    """Weight rows or tokens within a tile of 2^32: the last tile's row numbers would wrap."""
    import ctypes as C
    L, P = trmoe.lib(), C.c_void_p(256)
    most = (1 << 32) - 256

    def mat(rows):
        return C.byref(trmoe.I8Mat(256, 256, rows, 16, 1, 16, 0))

    def gemm(rows, m):
        return L.trk_gemm_i8(mat(rows), 0, P, 16, P, m, None, P, 0, 1 << 33, 0, None)

    def up(rows, m, slots):
        return L.trk_experts_up_i8(mat(rows), mat(rows), P, 16, P, m, P, P, slots, P, P, 1, 1 << 33, None)

    for rows, m, word in ((most + 1, 1, "rows"), ((1 << 32) - 1, 0, "rows"), (5, most + 1, "m (4294967041)"),
                          (5, (1 << 32) - 1, "m (4294967295)")):
        assert gemm(rows, m) == -1 and word in L.trk_last_error().decode()
    assert gemm(most, 0) == 0
    for rows, slots, ok in ((most, 16, True), (most, 17, False), (1 << 31, 32, True), ((1 << 31) + 1, 32, False)):
        assert up(rows, 0, slots) == (0 if ok else -1)
        assert ok or "too large" in L.trk_last_error().decode()
    assert L.trk_experts_down_i8(mat(most + 1), P, 16, P, 1, P, P, P, 1, None, None, P, 0, 1 << 33, 0, None) == -1
    assert "rows" in L.trk_last_error().decode()


def test_plan_extents_by_its_entries(tmp_path):
    import os
    import subprocess
    here = os.path.dirname(os.path.abspath(__file__))
    exe = str(tmp_path / "i8_plan_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", os.path.join(here, "i8_plan_check.cpp"), "-o", exe],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.startswith("ok"), r.stdout


def test_streams_of_other_devices_are_refused(monkeypatch):
    from types import SimpleNamespace
    trmoe._late()
    monkeypatch.setattr(trmoe, "_device", lambda: 0)
    assert trmoe._stream_here(SimpleNamespace(cuda_stream=5, device_index=0)) == 5
    with pytest.raises(trmoe.TrkError, match="a stream of device 1"):
        trmoe._stream_here(SimpleNamespace(cuda_stream=5, device_index=1))
