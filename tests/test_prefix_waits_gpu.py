"""The bounded waits of the tiled prefix, made to run out by a warp that withholds an arrival, without a fault: the call
returns, its rows are NaN, the status says why, and the next call gives what the one before gave."""

from __future__ import annotations

import time

import pytest
import torch

from tests.test_prefix_attention_gpu import build, on_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stall", [1, 2], ids=["queries", "weights"])
@pytest.mark.parametrize("b,h,prefix", [(40, 2, 200), (150, 2, 700), (20, 150, 1500)], ids=["one row tile", "two row tiles", "many tiles a CTA"])
@pytest.mark.parametrize("int8,dtype", [(False, torch.bfloat16), (False, torch.float32), (True, torch.bfloat16)], ids=["bf16", "bf16 to f32", "int8"])
@pytest.mark.parametrize("d", [64, 128])
def test_a_wait_that_runs_out_is_reported_and_poisons_only_that_call(d: int, int8: bool, dtype: torch.dtype, b: int, h: int, prefix: int, stall: int) -> None:
    from lazykv_b200 import _lib
    from lazykv_b200 import kernels as K

    K.status_attach()
    gen = torch.Generator().manual_seed(b)
    lens = [i % 4 for i in range(b)]
    cache, prefix_table, tables = build(gen, h, d, 32, int8, prefix, lens)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    query = torch.randn((b, 1, 2 * h, d), generator=gen).bfloat16().cuda()

    def call() -> tuple[torch.Tensor, torch.Tensor]:
        done = K.prefix_attention(query, pages, table, n, ptab, prefix, d**-0.5, scales=scales, out_dtype=dtype)
        torch.cuda.synchronize()
        return done

    want = call()
    assert K.device_status(clear=True) == 0
    K.status_poll(clear=True)
    K.debug_set(_lib.LKV_DEBUG_PREFIX_WAIT_NS, 1_000_000)
    K.debug_set(_lib.LKV_DEBUG_PREFIX_STALL_NEXT, stall)
    try:
        began = time.monotonic()
        out, lse = call()
        took = time.monotonic() - began
    finally:
        K.debug_set(_lib.LKV_DEBUG_PREFIX_STALL_NEXT, 0)
        K.debug_set(_lib.LKV_DEBUG_PREFIX_WAIT_NS, 2_000_000_000)
    assert K.status_poll(clear=False) == _lib.LKV_DEV_WAIT_TIMEOUT
    with pytest.raises(K.DeviceWaitError):
        K.raise_on_status("test")
    assert K.device_status(clear=True) == _lib.LKV_DEV_WAIT_TIMEOUT
    assert bool(out.isnan().all()) and bool(lse.isnan().all())
    assert took < 1.0  # a few waves of CTAs, a millisecond each
    again = call()
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    assert K.device_status(clear=True) == 0 and K.status_poll(clear=True) == 0
