"""What is left of a weight in the chunk attention: int8 pages 11 bits, however far value scales lie apart, as prefix_attention
keeps them of the same pages; and many turns of every ring in one CTA. Bounds: test_prefix_edges_gpu.near_pages (out is
bfloat16 here)."""

from __future__ import annotations

import pytest
import torch

from tests.test_prefix_attention_gpu import build, on_gpu
from tests.test_prefix_edges_gpu import SPREADS, near, near_pages, random_pages, rescale

pytestmark = pytest.mark.gpu


def attend(query: torch.Tensor, pages, scales, table, lens, ptab, prefix: int, scale: float):  # noqa: ANN001, ANN201
    """chunk_attention of chunks of equally many tokens [b, t, hq, d]."""
    from lazykv_b200 import kernels as K

    b, t = query.shape[:2]
    where = torch.arange(0, b * t + 1, t, dtype=torch.int32, device="cuda")
    out, lse = K.chunk_attention(query.cuda().flatten(0, 1), pages, table, lens, where, scale, scales=scales, prefix_table=ptab, prefix_len=prefix)
    assert K.device_status() == 0
    return out.view(query.shape), lse.view(query.shape[:3])


@pytest.mark.parametrize("t,g", [(1, 4), (6, 2), (50, 4)], ids=["a token", "one row tile", "two row tiles"])
@pytest.mark.parametrize("d", [64, 128])
def test_int8_weights_keep_eleven_bits(d: int, t: int, g: int) -> None:
    """Rows that see few tokens, whose values nearly cancel in many channels: the weights' rounding is what is left."""
    gen = torch.Generator().manual_seed(d + t)
    lens = [t + i % 3 for i in range(60)]
    cache, prefix_table, tables = build(gen, 2, d, 16, True, 2, lens, fill=0.0)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    query = torch.randn((60, t, 2 * g, d), generator=gen).bfloat16()
    out, lse = attend(query, pages, scales, table, n, ptab, 2, d**-0.5)
    near(cache, query, tables, lens, prefix_table, 2, d**-0.5, out, lse)


@pytest.mark.parametrize("spread", SPREADS, ids=str)
@pytest.mark.parametrize("b,t,h", [(3, 1, 2), (40, 1, 2), (2, 80, 2), (24, 70, 12)], ids=["parts of one row tile", "one row tile", "parts of two", "whole units"])
@pytest.mark.parametrize("d", [64, 128])
def test_int8_values_beside_far_larger_ones(d: int, b: int, t: int, h: int, spread) -> None:  # noqa: ANN001
    every, first, power, keys, all_of_them = spread
    gen = torch.Generator().manual_seed(b + power + d)
    prefix, lens = 700, [t + 3 + i % 9 for i in range(b)]
    cache, prefix_table, tables = build(gen, h, d, 32, True, prefix, lens, fill=0.0)
    # All keys point along one direction per head and queries too: scores around 25 with the keys as they are.
    along = torch.randn((1, h, d), generator=gen)
    k = (along + 0.1 * torch.randn((prefix, h, d), generator=gen)).bfloat16()
    cache.write(prefix_table, 0, k, torch.randn((prefix, h, d), generator=gen).bfloat16())
    cache.scales[:, :, 1] *= 2.0**all_of_them
    rescale(cache, prefix_table, prefix, every, first, 2.0**power, keys)
    if keys == 0.0:
        cache.scales[:, :, 0] = 0.0
    query = (along.transpose(0, 1).expand(h, 2, d).reshape(1, 1, 2 * h, d) * 3 * 64**0.5 / d**0.5 + 0.1 * torch.randn((b, t, 2 * h, d), generator=gen)).bfloat16()
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    out, lse = attend(query, pages, scales, table, n, ptab, prefix, d**-0.5)
    near(cache, query, tables, lens, prefix_table, prefix, d**-0.5, out, lse)


@pytest.mark.parametrize("b,h,t,g", [(40, 37, 1, 1), (1, 148, 500, 1), (4, 16, 300, 4)], ids=["short chunks", "two row tiles", "long chunks"])
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
def test_many_tiles_in_one_cta(d: int, int8: bool, b: int, h: int, t: int, g: int) -> None:
    """Two hundred and sixty tiles a CTA, or some fifty: many turns of every ring. Scores grow and fall from tile to tile, so
    references move and outputs are rescaled; pages are missing here and there, and the last tiles are not full."""
    gen = torch.Generator(device="cuda").manual_seed(b + d)
    bs, prefix, own = 64, 13 * 128 + 37, 1500
    pcols, cols = -(-prefix // bs), -(-own // bs)
    pages, scales = random_pages(gen, pcols + b * cols, h, bs, d, int8)
    order = torch.randperm(pcols + b * cols, generator=gen, device="cuda").to(torch.int32)
    ptab, table = order[:pcols].contiguous(), order[pcols:].view(b, cols).clone()
    for turn in range(7):  # keys of some pages larger
        (pages if scales is None else scales)[turn::7, :, 0] *= 2.0 ** (turn - 2)
    ptab[5], table[:, 3] = -1, -1
    lens = [max(t, own - 41 * i) for i in range(b)]
    query = torch.randn((b, t, h * g, d), generator=gen, device="cuda").bfloat16()
    out, lse = attend(query, pages, scales, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), ptab, prefix, d**-0.5)
    near_pages(pages, scales, query, table.tolist(), lens, ptab.tolist(), prefix, d**-0.5, out, lse)
