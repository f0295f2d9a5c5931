"""The bounded waits of the attention sums, made to run out by a warp that withholds an arrival, in every CTA or in one alone:
the call returns, a token that lost weights to it is NaN and every other one right, the status says why, and the next call is
right."""

from __future__ import annotations

import pytest
import torch

from tests.test_prefix_attention_gpu import build, on_gpu

pytestmark = pytest.mark.gpu

QUERIES, SCORES = 1, 2  # what is withheld: a chunk's queries, the room of scores that were read


class _Stalled:
    """Calls under a wait bound of two milliseconds."""

    def __enter__(self):  # noqa: ANN204
        from lazykv_b200 import _lib as L
        from lazykv_b200 import kernels as K

        self.L, self.K = L, K
        K.status_attach()
        assert K.device_status(clear=True) == 0
        K.status_poll(clear=True)
        K.debug_set(L.LKV_DEBUG_SUMS_WAIT_NS, 2_000_000)
        return self

    def call(self, which: int, cta: int, fn):  # noqa: ANN001, ANN201
        self.K.debug_set(self.L.LKV_DEBUG_SUMS_STALL_CTA, cta)
        self.K.debug_set(self.L.LKV_DEBUG_SUMS_STALL_NEXT, which)
        got = fn()
        torch.cuda.synchronize()
        return got, self.K.device_status(clear=True)

    def __exit__(self, *_) -> None:  # noqa: ANN002
        self.K.debug_set(self.L.LKV_DEBUG_SUMS_STALL_NEXT, 0)
        self.K.debug_set(self.L.LKV_DEBUG_SUMS_STALL_CTA, -1)
        self.K.debug_set(self.L.LKV_DEBUG_SUMS_WAIT_NS, 2_000_000_000)
        self.K.status_poll(clear=True)


def _case(d: int, int8: bool, new: list[int], lens: list[int]):  # noqa: ANN202
    from lazykv_b200 import kernels as K

    gen = torch.Generator().manual_seed(d + sum(new))
    cache, prefix_table, tables = build(gen, 2, d, 16, int8, 0, lens)
    pages, scales, _, table, n = on_gpu(cache, prefix_table, tables, lens)
    where = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    q = torch.randn((sum(new), 8, d), generator=gen).bfloat16().cuda()
    _, lse = K.chunk_attention(q, pages, table, n, where, d**-0.5, scales=scales)
    sums = torch.rand((len(lens), 2, table.shape[1] * 16), generator=gen).cuda()

    def call(out: torch.Tensor | None = None) -> torch.Tensor:
        """In place (the sums of earlier steps, copied), or into `out`."""
        given = sums.clone()
        return K.attention_sums(q, lse, pages, table, n, where, d**-0.5, sums=given, scales=scales, out=given if out is None else out)

    return call, sums


# New tokens and lengths: few rows (whole tiles, several a CTA); long chunks (tiles that several CTAs have chunks of).
CASES = [([1, 3, 2, 0], [40000, 30000, 50000, 300]), ([300, 33], [9000, 7000])]


@pytest.mark.parametrize("which", [QUERIES, SCORES], ids=["queries", "scores"])
@pytest.mark.parametrize(("new", "lens"), CASES, ids=["few rows", "long chunks"])
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
def test_one_cta_that_gives_up(d: int, int8: bool, new: list[int], lens: list[int], which: int) -> None:
    call, sums = _case(d, int8, new, lens)
    want = call()
    assert not bool(want.isnan().any())
    lost = 0
    with _Stalled() as stalled:
        for cta in range(0, 148, 3):
            out = torch.full_like(sums, 7.0) if cta % 2 else None
            got, status = stalled.call(which, cta, lambda: call(out))  # noqa: B023
            bad = got.isnan()
            assert bool((bad | (got == want)).all()), (cta, (~bad & (got != want)).nonzero()[:3].tolist())
            assert status == int(bad.any()), (cta, status)
            lost += int(bad.any())
    assert lost >= 20  # (CTAs without work, or with too few jobs to run out of room, lose nothing)
    assert torch.equal(call(), want)


@pytest.mark.parametrize(("new", "lens"), CASES, ids=["few rows", "long chunks"])
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_every_cta_gives_up(int8: bool, new: list[int], lens: list[int]) -> None:
    call, sums = _case(128, int8, new, lens)
    want = call()
    with _Stalled() as stalled:
        for out in (None, torch.full_like(sums, 7.0)):
            got, status = stalled.call(QUERIES, -1, lambda: call(out))  # noqa: B023
            assert status == 1
            for b, n in enumerate(lens):
                lost = n if new[b] else 0
                assert bool(got[b, :, :lost].isnan().all()), b
                assert torch.equal(got[b, :, lost:], want[b, :, lost:]), b  # what no query sees goes on, what no token has is 0
    assert torch.equal(call(), want)
