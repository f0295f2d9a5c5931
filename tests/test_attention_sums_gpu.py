"""The weights that cached tokens got, against their definition in 64 bits.

A weight is off by a factor within e^(+-e), e = (d + 5) 2^-24 reach (the score's float32 sum, with the scales), c 2^-20 of a
capped score, 2^-24 |lse| and |score| twice (the subtraction and the turn into the log2 domain) and the exponential's 2^-22;
a float32 sum of n weights and what was there before by (n + 2) 2^-24 of it. exp underflows below 2^-126, to at most so much
each."""

from __future__ import annotations

import math

import pytest
import torch

from tests import chunk_plain as P
from tests.test_chunk_attention_gpu import CASES, _kernels, _offsets
from tests.test_prefix_attention_gpu import build, on_gpu

pytestmark = pytest.mark.gpu


def definition(cache, query, lse, tables, lens, offsets, scale, cap, sums, last):  # noqa: ANN001, ANN201
    """(sums, bound) in float64."""
    batch, h, slots = sums.shape
    out, bound = torch.zeros(sums.shape, dtype=torch.float64), torch.zeros(sums.shape, dtype=torch.float64)
    d = query.shape[2]
    for b in range(batch):
        n = offsets[b + 1] - offsets[b]
        seen = max(0, min(lens[b], slots, len(tables[b]) * cache.bs))
        old = max(0, min(lens[b] - n, seen))
        out[b, :, :old] = sums[b, :, :old]
        if n and seen:
            z, size, _, see = P.scores(cache, query, b, tables, lens, offsets, [], 0, scale, cap)
            of = lse[offsets[b] : offsets[b + 1]].double()[..., None]
            live = see[:, None] & ~torch.isneginf(of)
            if last is not None:
                live[: max(0, n - last)] = False
            w = torch.where(live, torch.exp(z - of), 0.0)
            e = (d + 5) * 2.0**-24 * size + cap * 2.0**-20 + 2.0**-22 + torch.where(live, 3 * 2.0**-24 * (of.abs() + z.abs() + 1), 0.0)
            got = w.reshape(n, h, -1, w.shape[-1]).sum((0, 2))
            off = (w * torch.expm1(e)).nan_to_num(0.0).reshape(n, h, -1, w.shape[-1]).sum((0, 2))
            rows = n * query.shape[1] // h
            out[b, :, :seen] += got[:, :seen]
            bound[b, :, :seen] += off[:, :seen] + (rows + 2) * 2.0**-24 * out[b, :, :seen].abs().nan_to_num(0.0) + rows * 2.0**-126
        bound[b] += 2.0**-23 * out[b].abs().nan_to_num(0.0)
    return out, bound


def check(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor) -> None:
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    bad = ((got - want).abs() > bound) & ~want.isnan()
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), want[bad][:4].tolist())


@pytest.mark.parametrize("case", CASES, ids=lambda c: "h%d-g%d-p%d-L%d-b%d" % (c[0], c[1], c[2], c[3], len(c[4])))
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
def test_matches_the_definition(d: int, int8: bool, case) -> None:  # noqa: ANN001
    K = _kernels()
    h, g, bs, prefix, new, lens = case
    gen = torch.Generator().manual_seed(sum(lens) + prefix + d)
    cache, prefix_table, tables = build(gen, h, d, bs, int8, prefix, lens)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    offsets = _offsets(new)
    query = (1.5 * torch.randn((offsets[-1] + 2, h * g, d), generator=gen)).bfloat16()
    where, q = torch.tensor(offsets, dtype=torch.int32, device="cuda"), query.cuda()
    slots = table.shape[1] * bs - (5 if d == 64 else 0)
    before = torch.exp(torch.randn((len(lens), h, slots), generator=gen))
    before[:, 0, ::7] = 0.0
    for cap, last, sums in ((0.0, None, before), (20.0, 3, None)):
        lse = torch.full((query.shape[0], h * g), 3.0, device="cuda")
        K.chunk_attention(q, pages, table, n, where, d**-0.5, scales=scales, prefix_table=ptab, prefix_len=prefix, cap=cap, lse=lse)
        given = None if sums is None else sums.cuda()
        out = torch.full((len(lens), h, slots), 7.0, device="cuda") if sums is None else given
        got = K.attention_sums(q, lse, pages, table, n, where, d**-0.5, sums=given, last=last, cap=cap, scales=scales, out=out)
        assert got is out and K.device_status() == 0
        check(got, *definition(cache, query, lse.cpu(), tables, lens, offsets, d**-0.5, cap, torch.zeros_like(before) if sums is None else sums, last))
        if sums is not None:  # the same to the last bit, not in place too
            again = K.attention_sums(q, lse, pages, table, n, where, d**-0.5, sums=sums.cuda(), last=last, cap=cap, scales=scales)
            assert torch.equal(again, got)


def test_all_weights_sum_to_the_rows() -> None:
    """Without a prefix every row's weights sum to one."""
    K = _kernels()
    h, g, d, bs = 2, 4, 128, 16
    new, lens = [70, 5], [700, 5]
    gen = torch.Generator().manual_seed(1)
    cache, prefix_table, tables = build(gen, h, d, bs, True, 0, lens)
    pages, scales, _, table, n = on_gpu(cache, prefix_table, tables, lens)
    where = torch.tensor(_offsets(new), dtype=torch.int32, device="cuda")
    q = torch.randn((75, h * g, d), generator=gen).bfloat16().cuda()
    _, lse = K.chunk_attention(q, pages, table, n, where, d**-0.5, scales=scales)
    got = K.attention_sums(q, lse, pages, table, n, where, d**-0.5, scales=scales)
    assert got.shape == (2, h, table.shape[1] * bs)
    want = torch.tensor(new, dtype=torch.float64)[:, None].expand(2, h) * g
    assert math.isclose(float((got.double().cpu().sum(-1) - want).abs().max()), 0.0, abs_tol=280 * 2.0**-15)
