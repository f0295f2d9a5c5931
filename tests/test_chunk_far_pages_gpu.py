"""The packed operators on a cache whose pages lie past 2^32 bytes: the same, bit for bit, as on a small
cache that holds the same tokens."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_far_pages(int8: bool) -> None:
    from lazykv_b200 import kernels as K

    h, g, d, bs, b, own, new = 8, 2, 128, 64, 2, 600, 70
    cols = -(-own // bs)
    n = (2**32 // (h * 2 * bs * d * (1 if int8 else 2))) + 3 * b * cols
    gen = torch.Generator(device="cuda").manual_seed(1)
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, where = i32([own, own - 13]), i32([0, new, 2 * new])
    q = torch.randn((2 * new, h * g, d), generator=gen, device="cuda").bfloat16()
    k, v = (torch.randn((2 * new, h, d), generator=gen, device="cuda").bfloat16() for _ in range(2))
    kv = torch.randn((2, b, own, h, d), generator=gen, device="cuda").bfloat16()
    positions, freq = torch.arange(2 * new, dtype=torch.int32, device="cuda") + own, torch.full((64,), 0.1, device="cuda")
    got = []
    for pages_of, first in ((b * cols, 0), (n, n - b * cols)):
        pages = torch.empty((pages_of, h, 2, bs, d), dtype=torch.int8 if int8 else torch.bfloat16, device="cuda")
        scales = torch.empty((pages_of, h, 2, bs), device="cuda") if int8 else None
        table = (torch.arange(b * cols, dtype=torch.int32, device="cuda") + first).view(b, cols)
        K.paged_write(*kv, pages, table, i32([0, 0]), scales=scales)
        turned = K.paged_write_rotated(q, k, v, positions, freq, pages, table, lens, where, scales=scales)
        out, lse = K.chunk_attention(turned, pages, table, lens, where, 0.1, scales=scales, prefix_table=table[1].contiguous(), prefix_len=300)
        sums = K.attention_sums(turned, lse, pages, table, lens, where, 0.1, scales=scales)
        at = torch.arange(cols * bs, dtype=torch.int32, device="cuda").expand(b, h, -1).contiguous()
        left, sums2, at2 = K.paged_evict(pages, table, lens, sums, at, 100, scales=scales)
        back = K.paged_read(pages, table, i32([0, 0]), own, scales=scales)
        got.append([turned, out, lse, sums, left, sums2, at2, *back])
        del pages, scales
    assert all(torch.equal(x, y) for x, y in zip(*got))
    assert K.device_status() == 0
