"""What lies in a CTA's shared memory in the place of a page that is not there has no part in a result: to the last bit the
same, whatever ran before."""

from __future__ import annotations

import pytest
import torch

from tests.test_chunk_attention_gpu import _kernels
from tests.test_prefix_attention_gpu import build, on_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 40], ids=["one token", "two row tiles"])
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("d", [64, 128])
def test_earlier_calls_leave_nothing_in_missing_pages(d: int, cap: float, int8: bool, new: int) -> None:
    K = _kernels()
    batch, h, g, held = 90, 2, 4, 128 - new
    gen = torch.Generator().manual_seed(3)
    lens = [held + new] * batch
    cache, prefix_table, tables = build(gen, h, d, 16, int8, 0, lens)
    pages, scales, _, full, n = on_gpu(cache, prefix_table, tables, lens)
    table = full.clone()
    table[:, 2:5] = -1
    where = torch.arange(0, batch * new + 1, new, dtype=torch.int32, device="cuda")
    q = torch.randn((batch * new, h * g, d), generator=gen).bfloat16().cuda()

    def after(fill: int) -> list[torch.Tensor]:
        """Both operators, each behind a call of its own kind whose keys all hold `fill`."""
        before = torch.full_like(pages, fill)
        ones = None if scales is None else torch.ones_like(scales)
        _, l = K.chunk_attention(q, before, full, n, where, d**-0.5, scales=ones, cap=cap)  # noqa: E741
        out, lse = K.chunk_attention(q, pages, table, n, where, d**-0.5, scales=scales, cap=cap)
        K.attention_sums(q, l, before, full, n, where, d**-0.5, scales=ones, cap=cap)
        sums = K.attention_sums(q, lse, pages, table, n, where, d**-0.5, scales=scales, cap=cap)
        return [out, lse, sums]

    for _ in range(3):
        for x, y in zip(after(0), after(127)):
            assert torch.equal(x, y), int((x != y).sum())
    assert K.device_status() == 0
