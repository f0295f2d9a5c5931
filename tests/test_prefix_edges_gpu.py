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
