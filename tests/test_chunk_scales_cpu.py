"""Softmax scales and caps whose products leave float32 are refused: their scores would be NaN, or off by more than a rounding."""

from __future__ import annotations

import pytest

from lazykv_b200 import _lib as L
from tests.test_chunk_cpu import BASE, CHUNK, SUMS, _fields, lib  # noqa: F401


@pytest.mark.parametrize(("entry", "layout", "names", "cap_name"), [("lkv_chunk_attention", L.CHUNK_ARGS, CHUNK, "cap"), ("lkv_attention_sums", L.SUMS_ARGS, SUMS, "cap_scores")])
@pytest.mark.parametrize(("scale", "cap", "fine"), [
    (0.125, 0.0, True), (-0.125, 50.0, True), (0.0, 50.0, True), (1e-30, 7.0, True), (2e38, 0.0, True), (0.125, 1e36, True), (1e3, 1e-30, True),
    (3e38, 0.0, False),      # times log2(e)
    (-3e38, 0.0, False),
    (0.125, 1.3e38, False),  # 2 log2(e) times the cap
    (0.125, 3e38, False),
    (10.0, 1e-38, False),    # 2 log2(e) times their quotient
    (-3e38, 1.0, False),
    (1e-6, 1e35, False),     # a quotient below the normal numbers
])
def test_scales_and_caps(lib, entry: str, layout, names: list[str], cap_name: str, scale: float, cap: float, fine: bool) -> None:  # noqa: ANN001, F811
    # A call that would go on has too small a workspace: nothing reaches a device.
    make = _fields(layout, {**BASE, "cap": 0.0 if cap_name == "cap" else BASE["cap"], "workspace_bytes": 0}, names)
    code = getattr(lib, entry)(make(**{"scale": scale, cap_name: cap}), None)
    if fine:
        assert code == 4 and "needed" in L.last_error(), L.last_error()
    else:
        assert code == 1 and "scale" in L.last_error() and "cap" in L.last_error(), L.last_error()
