"""Shared-prefix attention where lengths, values and lists are at their edges, against the header's definition in
64 bits (`attend` below, in which a length is the caller's number whatever the table holds)."""

from __future__ import annotations

import math

import pytest
import torch

from tests.paged_plain import Cache
from tests.test_prefix_attention_gpu import build, on_gpu

pytestmark = pytest.mark.gpu


def attend(cache: Cache, query: torch.Tensor, tables: list[list[int]], lens: list[int], prefix_table: list[int], prefix_len: int,
           scale: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(out, lse, mass, reach) in float64: query t of sequence b sees the prefix and own tokens 0 .. lens[b] - T + t, those
    of them that have a page; mass = sum p |v| / sum p, reach = the largest sum |q k| scale of a row."""
    b, t, hq, d = query.shape
    h = cache.pages.shape[1]
    q = query.double().cpu()
    out, mass = torch.zeros((b, t, hq, d), dtype=torch.float64), torch.zeros((b, t, hq, d), dtype=torch.float64)
    lse, reach = torch.full((b, t, hq), -math.inf, dtype=torch.float64), torch.zeros((b, t, hq), dtype=torch.float64)
    kp, vp, okp = cache.read(prefix_table, list(range(prefix_len)))
    for i in range(b):
        room = len(tables[i]) * cache.bs  # no token past the table has a page
        ko, vo, oko = cache.read(tables[i], list(range(room)))
        for step in range(t):
            m = min(room, max(0, lens[i] - t + step + 1))
            k, v = torch.cat([kp[okp], ko[:m][oko[:m]]]), torch.cat([vp[okp], vo[:m][oko[:m]]])
            if k.shape[0] == 0:
                continue
            rows = q[i, step].view(h, hq // h, d)
            s = torch.einsum("hgd,nhd->hgn", rows, k) * scale
            reach[i, step] = (torch.einsum("hgd,nhd->hgn", rows.abs(), k.abs()) * abs(scale)).amax(-1).reshape(hq)
            lse[i, step] = torch.logsumexp(s, -1).reshape(hq)
            p = torch.softmax(s, -1)
            out[i, step] = torch.einsum("hgn,nhd->hgd", p, v).reshape(hq, d)
            mass[i, step] = torch.einsum("hgn,nhd->hgd", p, v.abs()).reshape(hq, d)
    return out, lse, mass, reach


def near(cache: Cache, query: torch.Tensor, tables, lens, prefix_table, prefix: int, scale: float, out: torch.Tensor, lse: torch.Tensor) -> None:
    """out (float32) and lse within what a weight's one rounding to bfloat16 or f16 and the scores' float32 sums leave
    (tests/test_prefix_attention_gpu.py derives the terms): 2^-8 of sum p |v|, and 2 (d + 4) 2^-24 reach and n 2^-24 of it."""
    want, wlse, mass, reach = attend(cache, query, tables, lens, prefix_table, prefix, scale)
    n = prefix + max(len(t) for t in tables) * cache.bs
    sums = (query.shape[-1] + 4) * 2.0**-24 * reach + 2.0**-22 + n * 2.0**-24
    err, lerr = (out.double().cpu() - want).abs(), (lse.double().cpu() - wlse).abs()
    bound = (2.0**-8 + 2 * sums[..., None]) * mass + 2.0**-23 * want.abs()
    empty = wlse == -math.inf
    assert bool((err <= bound).all()), float((err / bound.clamp_min(1e-30)).max())
    assert bool((lse.cpu()[empty] == -math.inf).all())
    assert bool((lerr <= sums + 4 * 2.0**-24 * (wlse.abs() + 1))[~empty].all()), float(lerr[~empty].max())


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("b,t,g", [(2, 4, 1), (7, 5, 4)])
def test_several_queries_of_a_length_past_the_table(b: int, t: int, g: int, int8: bool) -> None:
    """Lengths around the table's reach and far past it: tokens past the table are not there, and a query's sight is
    counted from the length as given, not from what the table holds."""
    from lazykv_b200 import kernels as K

    h, d, bs, prefix = 2, 64, 16, 21
    gen = torch.Generator().manual_seed(b)
    cache, prefix_table, tables = build(gen, h, d, bs, int8, prefix, [32] * b)
    lens = [34, 32 + t, 31, 32, 33, 2**31 - 1, -(2**31)][:b]
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    query = torch.randn((b, t, h * g, d), generator=gen).bfloat16()
    out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, prefix, d**-0.5, scales=scales, out_dtype=torch.float32)
    near(cache, query, tables, lens, prefix_table, prefix, d**-0.5, out, lse)


def near_int8(cache: Cache, query: torch.Tensor, tables, lens, prefix_table, prefix: int, scale: float, out: torch.Tensor, lse: torch.Tensor) -> None:
    """int8 pages, each row on its own: a weight times its value's scale is rounded to f16 once, 2^-11 of it or 2^-25
    of a unit of which the row's largest such product has 2^6 at least: n keys, codes up to 127, make that at most
    n 2^-31 top, top = max p max |v| / sum p over the row's keys. The rest as in `near`, with four more float32 roundings."""
    want, wlse, mass, reach = attend(cache, query, tables, lens, prefix_table, prefix, scale)
    b, t, hq, d = query.shape
    h = cache.pages.shape[1]
    n = prefix + max(len(x) for x in tables) * cache.bs
    kp, vp, okp = cache.read(prefix_table, list(range(prefix)))
    top = torch.zeros((b, t, hq), dtype=torch.float64)
    for i in range(b):
        ko, vo, oko = cache.read(tables[i], list(range(len(tables[i]) * cache.bs)))
        for step in range(t):
            m = min(ko.shape[0], max(0, lens[i] - t + step + 1))
            k, v = torch.cat([kp[okp], ko[:m][oko[:m]]]), torch.cat([vp[okp], vo[:m][oko[:m]]])
            if k.shape[0] > 0:
                p = torch.softmax(torch.einsum("hgd,nhd->hgn", query[i, step].double().cpu().view(h, hq // h, d), k) * scale, -1)
                top[i, step] = (p * v.abs().amax(-1).T[:, None]).amax(-1).reshape(hq)
    sums = (d + 4) * 2.0**-24 * reach + 2.0**-22 + n * 2.0**-24
    bound = (2.0**-11 + 2 * sums[..., None] + 4 * 2.0**-24) * mass + n * 2.0**-31 * top[..., None] + 2.0**-23 * want.abs()
    err, lerr = (out.double().cpu() - want).abs(), (lse.double().cpu() - wlse).abs()
    empty = wlse == -math.inf
    assert bool((err <= bound).all()), float((err / bound.clamp_min(1e-300)).max())
    assert bool((lerr <= sums + 4 * 2.0**-24 * (wlse.abs() + 1))[~empty].all()), float(lerr[~empty].max())


def rescale(cache: Cache, prefix_table: list[int], prefix: int, every: int, first: int, values: float, keys: float) -> None:
    """Every `every`-th token of the prefix from `first` on: values times `values`, keys times `keys` (powers of two, or 0)."""
    for pos in range(first, prefix, every):
        page, at = prefix_table[pos // cache.bs], pos % cache.bs
        cache.scales[page, :, 1, at] = (cache.scales[page, :, 1, at].double() * values).float()  # (2^170 is no float32)
        cache.scales[page, :, 0, at] *= keys


# Some tokens' values are many powers of two times the others', (every, first, power, what their keys are multiplied
# with, power of all values): with the others' weights (keys as they are, or all zero: one score for all), far less (a
# score some tens lower: negated keys of a query that points along them), from the first token on or late in the list.
SPREADS = [(50, 0, 20, 1.0, 0), (50, 49, 40, 1.0, 0), (13, 5, -20, 1.0, 0), (200, 7, 27, -1.0, 0), (200, 150, 27, -1.0, 0), (64, 63, 60, -1.0, 0),
           (5, 3, 100, 0.0, 0), (7, 2, -60, 0.0, 0), (90, 80, 170, 0.0, -60), (90, 0, 170, 0.0, -60)]


def spread_case(b: int, d: int, spread, bs: int, prefix: int, h: int = 2):  # noqa: ANN001, ANN201
    every, first, power, keys, all_of_them = spread
    gen = torch.Generator().manual_seed(b + power + d)
    lens = [3 + i % 9 for i in range(b)]
    cache, prefix_table, tables = build(gen, h, d, bs, True, prefix, lens, fill=0.0)
    # All keys point along one direction per head and queries too: scores around 25 with the keys as they are.
    along = torch.randn((1, h, d), generator=gen)
    k = (along + 0.1 * torch.randn((prefix, h, d), generator=gen)).bfloat16()
    cache.write(prefix_table, 0, k, torch.randn((prefix, h, d), generator=gen).bfloat16())
    cache.scales[:, :, 1] *= 2.0**all_of_them
    rescale(cache, prefix_table, prefix, every, first, 2.0**power, keys)
    if keys == 0.0:
        cache.scales[:, :, 0] = 0.0
    query = (along.transpose(0, 1).expand(h, 2, d).reshape(1, 1, 2 * h, d) * 3 * 64**0.5 / d**0.5 + 0.1 * torch.randn((b, 1, 2 * h, d), generator=gen)).bfloat16()
    return cache, prefix_table, tables, lens, query


@pytest.mark.parametrize("spread", SPREADS, ids=str)
@pytest.mark.parametrize("d", [64, 128])
def test_int8_values_beside_far_larger_ones_in_the_stream(d: int, spread) -> None:  # noqa: ANN001
    from lazykv_b200 import kernels as K

    cache, prefix_table, tables, lens, query = spread_case(3, d, spread, 16, 400)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, 400, d**-0.5, scales=scales, out_dtype=torch.float32)
    near_int8(cache, query, tables, lens, prefix_table, 400, d**-0.5, out, lse)
