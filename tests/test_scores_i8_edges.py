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
