"""The bounded waits of the chunk attention, made to run out in every CTA or in one alone: a row is NaN, or was not written, or is
right, whatever the workspace held, and the next call is right."""

from __future__ import annotations

import pytest
import torch

from tests.test_prefix_attention_gpu import build, on_gpu

pytestmark = pytest.mark.gpu

QUERIES, WEIGHTS = 1, 2  # what is withheld
SENTINEL = 7.0


# Units of one row tile and of two, pieces of the line that hold parts of several units, and whole ones.
@pytest.mark.parametrize(("new", "lens", "prefix"), [([300, 5], [9000, 5], 0), ([20, 3, 64, 1], [2900, 500, 1000, 700], 300), ([60] * 20, [60 + 40 * i for i in range(20)], 100)],
                         ids=["two row tiles", "one row tile", "short units"])
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_one_cta_that_gives_up(int8: bool, new: list[int], lens: list[int], prefix: int) -> None:
    from lazykv_b200 import _lib as L
    from lazykv_b200 import kernels as K

    K.status_attach()
    gen = torch.Generator().manual_seed(sum(new))
    cache, prefix_table, tables = build(gen, 2, 64, 16, int8, prefix, lens)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    q = torch.randn((sum(new), 8, 64), generator=gen).bfloat16().cuda()
    where = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    nbytes = L.lib().lkv_chunk_attention_workspace(q.shape[0], len(new), 8, 2, 64, prefix, table.shape[1] * 16)
    out, lse = torch.empty_like(q), torch.empty((q.shape[0], 8), device="cuda")

    def call() -> tuple[torch.Tensor, torch.Tensor]:
        out.fill_(SENTINEL)
        lse.fill_(SENTINEL)
        stale = torch.ones((nbytes + 1) // 2, dtype=torch.bfloat16, device="cuda")  # what the workspace will hold
        del stale
        K.chunk_attention(q, pages, table, n, where, 0.125, scales=scales, prefix_table=ptab, prefix_len=prefix, out=out, lse=lse)
        torch.cuda.synchronize()
        return out.clone(), lse.clone()

    want = call()
    assert K.device_status(clear=True) == 0 and not bool(want[0].isnan().any())
    K.status_poll(clear=True)
    lost = 0
    K.debug_set(L.LKV_DEBUG_CHUNK_WAIT_NS, 2_000_000)
    try:
        for cta in (*range(0, 148, 2), -1):
            for which in (QUERIES, WEIGHTS):
                K.debug_set(L.LKV_DEBUG_CHUNK_STALL_CTA, cta)
                K.debug_set(L.LKV_DEBUG_CHUNK_STALL_NEXT, which)
                got = call()
                status = K.device_status(clear=True)
                wrong = False
                for x, y in zip(got, want):
                    fine = x.isnan() | (x == SENTINEL) | (x == y)
                    assert bool(fine.all()), (cta, which, (~fine).nonzero()[:3].tolist())
                    wrong = wrong or bool((x.isnan() | (x == SENTINEL)).any())
                assert status == (L.LKV_DEV_WAIT_TIMEOUT if wrong else 0), (cta, which)
                lost += wrong
                if cta < 0:  # nobody has finished anything
                    assert bool((got[0].isnan() | (got[0] == SENTINEL)).all()) and bool((got[1].isnan() | (got[1] == SENTINEL)).all())
    finally:
        K.debug_set(L.LKV_DEBUG_CHUNK_STALL_NEXT, 0)
        K.debug_set(L.LKV_DEBUG_CHUNK_STALL_CTA, -1)
        K.debug_set(L.LKV_DEBUG_CHUNK_WAIT_NS, 2_000_000_000)
        K.status_poll(clear=True)
    assert lost >= 20
    again = call()
    assert all(torch.equal(x, y) for x, y in zip(again, want)) and K.device_status(clear=True) == 0
