"""Attention of packed chunks against its definition in 64 bits.

Bounds, per output element: a weight (times its value's scale) is rounded once to bfloat16, half a step of 2^-8 of it; a
score is a float32 sum of d products with up to four more roundings, off by delta = (d + 4) 2^-24 reach, reach the largest
sum |q k| scale of the row; a capped one further by c 2^-20 (the exponential's argument and result 2^-22 each, the quotient
2^-23, the last step's rounding 2^-24 of 2 c, all times c). Both move every weight by a factor within e^(+-); the exponential's
own error is 2^-22 and a reference rounded between passes 2^-22; float32 sums of n keys n 2^-24 at worst. An output is off by
(2^-8 + 2 (those)) mass, mass = sum p |v|, and half a bfloat16 step of itself; lse by those and float32's roundings of
its own size. A product of a code, its scale and a weight is rounded once more, 2^-24."""

from __future__ import annotations

import math

import pytest
import torch

from tests import chunk_plain as P
from tests.test_prefix_attention_gpu import build, on_gpu

pytestmark = pytest.mark.gpu


def _kernels():  # noqa: ANN202
    from lazykv_b200 import kernels

    return kernels


def _offsets(new: list[int]) -> list[int]:
    return [sum(new[:i]) for i in range(len(new) + 1)]


def check(cache, query, tables, lens, offsets, prefix_table, prefix, scale, cap, out, lse) -> None:  # noqa: ANN001
    want, wlse, mass, reach = P.attend(cache, query, tables, lens, offsets, prefix_table, prefix, scale, cap)
    out, lse, live = out.double().cpu(), lse.double().cpu(), offsets[-1]
    want, wlse, mass, reach, out, lse = want[:live], wlse[:live], mass[:live], reach[:live], out[:live], lse[:live]
    d, n = query.shape[-1], prefix + max(lens, default=0)
    sums = (d + 4) * 2.0**-24 * reach + cap * 2.0**-20 + 2.0**-21 + n * 2.0**-24
    bound = (2.0**-8 + 2.0**-23 + 2 * sums[..., None]) * mass + 2.0**-8 * want.abs() + 2.0**-120
    odd, lost = ~want.isfinite(), wlse.isnan()
    same = torch.where(want.isnan(), out.isnan(), out == want)
    assert bool(same[odd & ~lost[..., None]].all()), "infinities and NaN that are seen"
    err = (out - want).abs()
    assert bool((err <= bound)[~odd & ~lost[..., None]].all()), float((err / bound)[~odd & ~lost[..., None]].max())
    assert torch.equal(lse.isnan(), lost)
    empty = wlse == -math.inf
    assert bool((lse[empty] == -math.inf).all()) and bool((out[empty] == 0).all())
    fine = ~empty & ~lost
    lerr, lbound = (lse - wlse).abs()[fine], (sums + 4 * 2.0**-24 * (wlse.abs() + 1))[fine]
    assert bool((lerr <= lbound).all()), float((lerr / lbound).max())


CASES = [
    # heads, group, page, prefix, new tokens, own lengths
    (1, 1, 16, 0, [1], [1]),
    (2, 4, 16, 0, [17], [317]),
    (2, 4, 16, 100, [0, 1, 17, 40], [0, 1, 17, 300]),
    (1, 8, 32, 257, [3, 0, 200, 1, 1], [3, 70, 200, 128, 129]),
    (3, 7, 64, 0, [50, 1], [50, 513]),          # seven query heads a KV head: tokens that two row tiles share
    (1, 3, 16, 385, [171], [600]),              # 513 rows: a third block of one row
    (2, 1, 128, 128, [128, 256, 129], [128, 512, 129]),
    (1, 16, 16, 0, [40], [2000]),
    (8, 4, 16, 0, [300], [300]),                # a causal chunk without anything before it
    (1, 4, 64, 3000, [33] * 12, [33 + 50 * i for i in range(12)]),
    (1, 40, 16, 17, [5, 2], [5, 900]),          # 40 query heads a KV head
    (4, 2, 16, 0, [1] * 300, [1 + (7 * i) % 190 for i in range(300)]),  # more units than CTAs
    (8, 1, 16, 0, [1] * 40, [1000 + 9 * i for i in range(40)]),                       # many tiles a CTA, all of few rows
    (8, 1, 16, 40, [1] * 30 + [140], [1000 + 9 * i for i in range(30)] + [1400]),  # and one unit of two row tiles among them
    (1, 1, 16, 0, [2, 3], [1, 0]),              # chunks longer than what their sequences hold: rows that see nothing
]


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
    rows = offsets[-1] + 3
    query = (1.5 * torch.randn((rows, h * g, d), generator=gen)).bfloat16()
    for cap in (0.0, 20.0):
        out = torch.full((rows, h * g, d), 7.0, dtype=torch.bfloat16, device="cuda")
        lse = torch.full((rows, h * g), 7.0, device="cuda")
        got = K.chunk_attention(query.cuda(), pages, table, n, torch.tensor(offsets, dtype=torch.int32, device="cuda"), d**-0.5, scales=scales, prefix_table=ptab,
                                prefix_len=prefix, cap=cap, out=out, lse=lse)
        assert got[0] is out and got[1] is lse
        assert K.device_status() == 0
        assert bool((out[-3:] == 7.0).all()) and bool((lse[-3:] == 7.0).all()), "rows of no sequence are left as they were"
        check(cache, query, tables, lens, offsets, prefix_table, prefix, d**-0.5, cap, out, lse)
