"""The test hooks of the attention sums' and the chunk attention's bounded waits take no value outside their range."""

from __future__ import annotations

import ctypes

import pytest

from lazykv_b200 import _lib as L


@pytest.mark.parametrize(("key", "values", "says"), [
    (L.LKV_DEBUG_SUMS_WAIT_NS, (0, -1, 2_000_000_001), "sums wait bound"),
    (L.LKV_DEBUG_SUMS_STALL_NEXT, (-1, 3), "of the attention sums"),
    (L.LKV_DEBUG_SUMS_STALL_CTA, (-2, 2**31), "of the attention sums"),
    (L.LKV_DEBUG_CHUNK_STALL_CTA, (-2, 2**31), "of the chunk attention"),
])
def test_hooks_are_bounded(key: int, values: tuple[int, ...], says: str) -> None:
    if not L.LIB_PATH.exists():
        from lazykv_b200.build import build

        build()
    for value in values:
        assert L.lib().lkv_debug_set(key, ctypes.c_int64(value)) == 1 and says in L.last_error()
