"""The sizes that the GPU tests of the 4-bit products' kernels use take the kernels that they are meant for."""
from __future__ import annotations

import os
import subprocess

import mx4forms as S


def test_sizes_take_their_forms(tmp_path):
    here = os.path.dirname(os.path.abspath(__file__))
    exe = str(tmp_path / "mx4_forms_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", os.path.join(here, "mx4_forms_check.cpp"), "-o", exe], check=True)
    asked = [(f"gemm {m} {rows} {k}", form) for form, sizes in S.GEMMS.items() for m, rows, k in sizes]
    for op, sizes in (("up", S.UP), ("down", S.DOWN)):
        asked += [(f"{op} {m} {slots} {E} {rows}", form) for form, (m, slots, E, rows) in sizes.items()]
    got = subprocess.run([exe], input="\n".join(a for a, _ in asked), check=True, capture_output=True, text=True).stdout.split("\n")
    assert [(a, g) for (a, _), g in zip(asked, got)] == asked
    far = "\n".join(f"gemm {m} {rows} {k}" for m, rows, k in (S.FAR_X, S.FAR_W))
    assert "strip" not in subprocess.run([exe], input=far, check=True, capture_output=True, text=True).stdout
