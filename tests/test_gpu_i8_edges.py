"""The int8 products and the quantisation of rows at the ends of their arguments, on the GPU against their plain 64-bit forms
(tests/i8ref.py)."""
from __future__ import annotations

import pytest

import trmoe
from test_gpu_scores_i8 import say

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
