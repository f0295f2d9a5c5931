"""What the test hooks of the tiled prefix's waits refuse (include/lkv.h)."""

from __future__ import annotations

import pytest


@pytest.mark.parametrize("key,value", [(4, 0), (4, -1), (4, 2_000_000_001), (5, -1), (5, 3)])
def test_the_wait_hooks_refuse(key: int, value: int) -> None:
    from lazykv_b200 import _lib
    from lazykv_b200 import kernels as K

    if not _lib.LIB_PATH.exists():
        from lazykv_b200.build import build

        build()
    with pytest.raises(_lib.LkvError):
        K.debug_set(key, value)
    assert (_lib.LKV_DEBUG_PREFIX_WAIT_NS, _lib.LKV_DEBUG_PREFIX_STALL_NEXT) == (4, 5)
