"""Shared-prefix attention where lengths, values and lists are at their edges, against the header's definition in
64 bits (`attend` below, in which a length is the caller's number whatever the table holds)."""

from __future__ import annotations

import math

import pytest
import torch

from tests.paged_plain import Cache
from tests.test_prefix_attention_gpu import build, on_gpu

pytestmark = pytest.mark.gpu


def tokens(pages: torch.Tensor, scales: torch.Tensor | None, j: int, table: torch.Tensor, n: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Head j's keys and values [..., n, d] of the first n tokens of page lists `table` [..., columns] in float64, and which
    of them have a page."""
    bs = pages.shape[3]
    at = torch.arange(n, device=pages.device)
    ids = table.long()[..., at // bs]
    there = (ids >= 0) & (ids < pages.shape[0])
    take = torch.where(there, ids, 0)
    x = pages[take, j, :, at % bs].double()  # [..., n, 2, d]
    if scales is not None:
        x = x * scales[take, j, :, at % bs].double()[..., None]
    return x[..., 0, :], x[..., 1, :], there


def attend(query: torch.Tensor, pages: torch.Tensor, scales: torch.Tensor | None, tables: list[list[int]], lens: list[int], prefix_table: list[int], prefix_len: int,
           scale: float) -> tuple[torch.Tensor, ...]:
    """(out, lse, mass, reach, top) in float64: query t of sequence b sees the prefix and own tokens 0 .. lens[b] - T + t,
    those of them that have a page. mass = sum p |v| / sum p per output element; reach = the largest sum |q k| scale and
    top = the largest p max |v| / sum p of a row's keys."""
    b, t, hq, d = query.shape
    h, bs = pages.shape[1], pages.shape[3]
    g = hq // h
    table, ptab = torch.tensor(tables, device="cuda").view(b, -1), torch.tensor(prefix_table, device="cuda")
    room = table.shape[1] * bs  # no token past the table has a page
    sight = torch.tensor([[min(room, max(0, n - t + i + 1)) for i in range(t)] for n in lens], device="cuda")  # [b, t]
    unseen = torch.arange(room, device="cuda") >= sight[..., None]  # [b, t, room]
    q = query.cuda().double().view(b, t, h, g, d)
    out, mass = (torch.zeros((b, t, h, g, d), dtype=torch.float64, device="cuda") for _ in range(2))
    lse, reach, top = (torch.zeros((b, t, h, g), dtype=torch.float64, device="cuda") for _ in range(3))
    for j in range(h):
        kp, vp, okp = tokens(pages, scales, j, ptab, prefix_len)
        ko, vo, oko = tokens(pages, scales, j, table, room)
        rows = q[:, :, j]  # [b, t, g, d]
        gone = torch.cat([(~okp).expand(b, t, g, -1), (unseen | ~oko[:, None])[:, :, None].expand(b, t, g, room)], -1)
        vp, vo = torch.where(okp[:, None], vp, 0.0), torch.where((oko & ~unseen.all(1))[..., None], vo, 0.0)  # what no row sees may hold anything
        s = torch.cat([rows @ kp.T, torch.einsum("btgd,bnd->btgn", rows, ko)], -1) * scale
        size = torch.cat([rows.abs() @ kp.abs().T, torch.einsum("btgd,bnd->btgn", rows.abs(), ko.abs())], -1) * abs(scale)
        s = torch.where(gone, -math.inf, s)
        lse[:, :, j] = torch.logsumexp(s, -1)
        p = torch.where(gone, 0.0, torch.exp(s - torch.where(lse[:, :, j] == -math.inf, 0.0, lse[:, :, j])[..., None]))
        reach[:, :, j] = torch.where(gone, 0.0, size).amax(-1)
        p1, p2 = p[..., :prefix_len], p[..., prefix_len:]
        out[:, :, j] = p1 @ vp + torch.einsum("btgn,bnd->btgd", p2, vo)
        mass[:, :, j] = p1 @ vp.abs() + torch.einsum("btgn,bnd->btgd", p2, vo.abs())
        most = torch.cat([vp.abs().amax(-1).expand(b, -1), vo.abs().amax(-1)], -1)  # [b, keys]
        top[:, :, j] = (p * most[:, None, None]).amax(-1)
    return out.view(b, t, hq, d), lse.view(b, t, hq), mass.view(b, t, hq, d), reach.view(b, t, hq), top.view(b, t, hq)


def near(cache: Cache, *rest) -> None:  # noqa: ANN002
    near_pages(cache.pages.cuda(), None if cache.scales is None else cache.scales.cuda(), *rest)


def near_pages(pages: torch.Tensor, scales: torch.Tensor | None, query: torch.Tensor, tables, lens, prefix_table, prefix: int, scale: float,
               out: torch.Tensor, lse: torch.Tensor, queries: slice = slice(None)) -> None:
    """out and lse, of some of a step's queries, against `attend`. A score is a float32 sum of d products (two more roundings for the scales):
    off by at most delta = (d + 4) 2^-24 reach, which moves a weight by a factor within e^(+-delta); exp2 is off by 2^-22 and
    the sums over n keys by n 2^-24 at most. bf16 pages: a weight is rounded to bfloat16, 2^-8 of it, or, for a float32 output, has a second
    term for what is left: 2^-7 of it at most, less 2^-8 of that. int8 pages: a weight
    times its value's scale is rounded to f16, 2^-11 of it or 2^-25 of a unit of which the row's largest such product has
    2^6 at least; codes go up to 127, so n keys make that n 2^-31 top at most; four more float32 roundings. A bfloat16 output is rounded once more, 2^-8 of it."""
    want, wlse, mass, reach, top = attend(query, pages, scales, tables, lens, prefix_table, prefix, scale)
    n = prefix + max(len(x) for x in tables) * pages.shape[3]
    sums = (query.shape[-1] + 4) * 2.0**-24 * reach + 2.0**-22 + n * 2.0**-24
    fine = out.dtype == torch.float32
    if scales is not None:
        bound = (2.0**-11 + 2 * sums[..., None] + 4 * 2.0**-24) * mass + n * 2.0**-31 * top[..., None]
    else:
        bound = ((2.0**-15 if fine else 2.0**-8) + 2 * sums[..., None]) * mass
    bound = bound + (2.0**-23 if fine else 2.0**-8 * (1 + 2.0**-7)) * want.abs() + (0 if fine else 2.0**-8 * bound)
    want, wlse, bound, sums, out, lse = (x[:, queries] for x in (want, wlse, bound, sums, out, lse))
    empty = wlse == -math.inf
    err, lerr = (out.double() - want).abs(), (lse.double() - wlse).abs()
    assert bool((err <= bound).all()), float((err / bound.clamp_min(1e-300)).max())
    assert bool((lse[empty] == -math.inf).all())
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
    near(cache, query, tables, lens, prefix_table, 400, d**-0.5, out, lse)


@pytest.mark.parametrize("spread", SPREADS, ids=str)
@pytest.mark.parametrize("b,h", [(40, 2), (150, 1), (24, 160)], ids=["one row tile", "two row tiles", "several tiles of the prefix a CTA"])
@pytest.mark.parametrize("d", [64, 128])
def test_int8_values_beside_far_larger_ones_in_the_tiles(d: int, b: int, h: int, spread) -> None:  # noqa: ANN001
    from lazykv_b200 import kernels as K

    cache, prefix_table, tables, lens, query = spread_case(b, d, spread, 32, 700, h)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, 700, d**-0.5, scales=scales, out_dtype=torch.float32)
    near(cache, query, tables, lens, prefix_table, 700, d**-0.5, out, lse)
    assert K.device_status() == 0


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
def test_values_that_are_not_finite_in_many_sequences_last_tokens(d: int, int8: bool) -> None:
    """Every sequence's last token is infinite or NaN here and there: the queries before it get what they get with
    that token's row all zeros, at every place of a list's end in its stage."""
    from lazykv_b200 import kernels as K

    h, g, bs, t, b = 2, 4, 16, 3, 60
    gen = torch.Generator().manual_seed(d)
    lens = [t + i for i in range(b)]
    cache, prefix_table, tables = build(gen, h, d, bs, int8, 20, lens)
    for i, n in enumerate(lens):
        x = torch.randn((1, h, d), generator=gen).bfloat16()
        x[..., i % d] = (torch.inf, -torch.inf, torch.nan)[i % 3]
        cache.write(tables[i], n - 1, x, x)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    query = torch.randn((b, t, h * g, d), generator=gen).bfloat16()
    out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, 20, d**-0.5, scales=scales, out_dtype=torch.float32)
    zero = torch.zeros((1, h, d), dtype=torch.bfloat16)
    for i, m in enumerate(lens):
        cache.write(tables[i], m - 1, zero, zero)
    near(cache, query, tables, lens, prefix_table, 20, d**-0.5, out, lse, slice(0, t - 1))


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("b,prefix,at", [(2, 0, 5), (2, 300, 299), (2, 300, 5), (40, 300, 299), (40, 300, 5)])
def test_a_value_that_is_not_finite_counts_under_any_weight(b: int, prefix: int, at: int, int8: bool, bad: float) -> None:
    """A token that every row sees, whose score is hundreds below the others' (its weight is 0 in float32), has a value
    that is not finite: exp(-500) infinity is infinite in the definition, and no row is finite there, wherever the token
    lies: at a list's end or before, in the own tokens, the streamed prefix or the tiled one."""
    from lazykv_b200 import kernels as K

    d, bs, n_own = 64, 16, 9
    gen = torch.Generator().manual_seed(at)
    cache, prefix_table, tables = build(gen, 1, d, bs, int8, prefix, [n_own] * b)
    key, value = torch.full((1, 1, d), -8.0).bfloat16(), torch.randn((1, 1, d), generator=gen).bfloat16()
    value[..., 3] = bad
    for table in [prefix_table] if prefix else tables:
        cache.write(table, at, key, value)
        if int8:
            cache.pages[table[at // bs], 0, 0, at % bs], cache.scales[table[at // bs], 0, 0, at % bs] = -127, 8 / 127
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, [n_own] * b)
    query = torch.full((b, 1, 4, d), 8.0).bfloat16()
    out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, prefix, d**-0.5, scales=scales, out_dtype=torch.float32)
    assert not bool(out[..., 3].isfinite().any()) and bool(lse.isfinite().all())
    if not int8:  # (int8: one scale for the whole row)
        assert bool(out[..., :3].isfinite().all()) and bool(out[..., 4:].isfinite().all())


def random_pages(gen: torch.Generator, n: int, h: int, bs: int, d: int, int8: bool) -> tuple[torch.Tensor, torch.Tensor | None]:
    """A cache on the GPU, every row of it filled."""
    if not int8:
        return torch.randn((n, h, 2, bs, d), generator=gen, device="cuda").bfloat16(), None
    pages = torch.randint(-127, 128, (n, h, 2, bs, d), generator=gen, device="cuda", dtype=torch.int8)
    return pages, (0.5 + torch.rand((n, h, 2, bs), generator=gen, device="cuda")) / 64


@pytest.mark.parametrize("b,h,g,t", [(20, 148, 1, 1), (35, 148, 4, 1), (50, 74, 2, 3)], ids=["one row tile", "two row tiles", "several CTAs of rows"])
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["to f32", "to bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_many_tiles_of_the_prefix_in_one_cta(d: int, dtype: torch.dtype, int8: bool, b: int, h: int, g: int, t: int) -> None:
    """A CTA of rows per SM: each takes the whole prefix, 22 tiles, past two turns of every ring it has. Scores grow and
    fall from tile to tile, so references move and outputs are rescaled; some pages are missing, two tiles have none at
    all, and the last tile is not full."""
    from lazykv_b200 import kernels as K

    gen = torch.Generator(device="cuda").manual_seed(b + d)
    bs, prefix = 64, 21 * 128 + 37
    cols = -(-prefix // bs)
    pages, scales = random_pages(gen, cols + b + 2, h, bs, d, int8)
    order = torch.randperm(cols + b + 2, generator=gen, device="cuda").tolist()
    prefix_table, tables = order[:cols], [[x] for x in order[cols : cols + b]]
    for col in range(cols):  # (the first tile's scores are small)
        by = (0.25, 0.5, 4.0, 1.0, 8.0, 0.125, 16.0)[(col // 2) % 7]
        (pages if scales is None else scales)[prefix_table[col], :, 0] *= by
    for col in (5, 14, 15, 16, 17, 30):
        prefix_table[col] = -1 if col % 2 else len(pages) + col
    lens = [(7 * i) % 64 for i in range(b)]
    query = (1.5 * torch.randn((b, t, h * g, d), generator=gen, device="cuda")).bfloat16()
    out, lse = K.prefix_attention(query, pages, torch.tensor(tables, dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                  torch.tensor(prefix_table, dtype=torch.int32, device="cuda"), prefix, d**-0.5, scales=scales, out_dtype=dtype)
    assert out.dtype == dtype
    near_pages(pages, scales, query, tables, lens, prefix_table, prefix, d**-0.5, out, lse)
    assert K.device_status() == 0


@pytest.mark.parametrize("prefix", [0, 700])
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
def test_more_stages_of_the_stream_than_its_warps_hold(d: int, int8: bool, prefix: int) -> None:
    """Own tokens of 64 sequences, up to 2,000 and 4,000, some none: every warp that the GPU holds takes some thirty
    stages or more, past many turns of its ring, over several sequences; scores grow and fall along a list."""
    from lazykv_b200 import kernels as K

    gen = torch.Generator(device="cuda").manual_seed(prefix + d)
    b, h, g, t, bs, most = 64, 8, 2, 2, 32, 2000 if d == 128 else 4000
    cols, pcols = -(-most // bs), -(-prefix // bs)
    pages, scales = random_pages(gen, b * cols + pcols, h, bs, d, int8)
    order = torch.randperm(b * cols + pcols, generator=gen, device="cuda")
    for turn in range(5):
        (pages if scales is None else scales)[turn::7, :, 0] *= 2.0 ** (turn - 2)
    table, ptab = order[: b * cols].view(b, cols).int(), order[b * cols :].int()
    lens = [most - (977 * i + 5) % 500 if i % 9 else 0 for i in range(b)]
    query = (1.5 * torch.randn((b, t, h * g, d), generator=gen, device="cuda")).bfloat16()
    out, lse = K.prefix_attention(query, pages, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), ptab, prefix, d**-0.5, scales=scales,
                                  out_dtype=torch.float32)
    near_pages(pages, scales, query, table.tolist(), lens, ptab.tolist(), prefix, d**-0.5, out, lse)
    assert K.device_status() == 0


@pytest.mark.parametrize("b,prefix", [(2, 1000), (40, 1000), (5, 0)], ids=["streamed", "tiled", "own tokens"])
@pytest.mark.parametrize("d", [64, 128])
def test_a_float32_output_of_bf16_pages_has_the_bits_of_one(d: int, b: int, prefix: int) -> None:
    """All values of a channel are alike, so that a weight's rounding shows in the output as it is and no mean over keys
    hides it: 2^-15 of it and the float32 sums, where one bfloat16 term would leave up to 2^-8."""
    from lazykv_b200 import kernels as K

    gen = torch.Generator().manual_seed(d + b)
    lens = [30 + i for i in range(b)]
    cache, prefix_table, tables = build(gen, 2, d, 16, False, prefix, lens, fill=0.0)
    cache.pages[:, :, 1] = torch.linspace(-3, 5, d).bfloat16()
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    query = (2 * torch.randn((b, 1, 4, d), generator=gen)).bfloat16()
    out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, prefix, d**-0.5, out_dtype=torch.float32)
    near(cache, query, tables, lens, prefix_table, prefix, d**-0.5, out, lse)


@pytest.mark.parametrize("b", [2, 40])
def test_a_softmax_scale_of_zero_makes_any_queries_alike(b: int) -> None:
    """int8 pages, queries of 2^120 and more: every seen key has the same weight."""
    from lazykv_b200 import kernels as K

    gen = torch.Generator().manual_seed(b)
    lens = [5] * b
    cache, prefix_table, tables = build(gen, 1, 64, 16, True, 200, lens)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    query = (torch.randn((b, 1, 4, 64), generator=gen) * 2.0**122).bfloat16()
    out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, 200, 0.0, scales=scales, out_dtype=torch.float32)
    near(cache, query, tables, lens, prefix_table, 200, 0.0, out, lse)


@pytest.mark.parametrize("up,queries", [(126, -126), (-108, 108), (-108, 122), (108, 4)])
@pytest.mark.parametrize("b", [2, 40])
def test_int8_keys_and_queries_far_apart(b: int, up: int, queries: int) -> None:
    """Key scales times 2^up and queries times 2^queries under a softmax scale that makes ordinary scores of them: no
    product of two of the three, nor with the codes, passes float32's end on the way."""
    from lazykv_b200 import kernels as K

    gen = torch.Generator().manual_seed(b)
    lens = [5 + i % 7 for i in range(b)]
    cache, prefix_table, tables = build(gen, 1, 64, 16, True, 200, lens, fill=0.0)
    cache.scales[:, :, 0] = (cache.scales[:, :, 0].double() * 2.0**up).float()
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    query = (torch.randn((b, 1, 4, 64), generator=gen).double() * 2.0**queries).bfloat16()
    scale = 0.125 * 2.0 ** -(up + queries)
    out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, 200, scale, scales=scales, out_dtype=torch.float32)
    near(cache, query, tables, lens, prefix_table, 200, scale, out, lse)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["to f32", "to bf16"])
@pytest.mark.parametrize("b,prefix,at", [(2, 0, 5), (2, 0, 70), (2, 1000, 17), (2, 1000, 999), (40, 1000, 17), (40, 1000, 999), (150, 300, 40)])
def test_an_infinite_value_that_is_seen_makes_an_infinite_output(b: int, prefix: int, at: int, dtype: torch.dtype) -> None:
    """bf16 pages, one value infinite, of an ordinary weight: its channel is infinite with its sign, as in the definition,
    and the other channels are what they are without it. Values with few bits and equal scores make terms of zero likely."""
    from lazykv_b200 import kernels as K

    d, bs, n_own = 64, 16, 80
    gen = torch.Generator().manual_seed(at)
    cache, prefix_table, tables = build(gen, 1, d, bs, False, prefix, [n_own] * b)
    cache.pages[:, :, 0] = 0.0  # every score is zero, every weight the same power of two
    for table in [prefix_table] if prefix else tables:
        cache.pages[table[at // bs], 0, 1, at % bs, 3] = math.inf
        cache.pages[table[at // bs], 0, 1, at % bs, 40] = -math.inf
    query = torch.randn((b, 1, 4, d), generator=gen).bfloat16()
    for spread in (0.0, 0.3):
        if spread:
            cache.pages[:, :, 0] = (spread * torch.randn(cache.pages[:, :, 0].shape, generator=gen)).bfloat16()
        pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, [n_own] * b)
        out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, prefix, d**-0.5, out_dtype=dtype)
        assert bool((out[..., 3] == math.inf).all()) and bool((out[..., 40] == -math.inf).all())
        plain = Cache(1, 1, bs, d, False)
        plain.pages = cache.pages.clone()
        plain.pages[:, :, 1, :, [3, 40]] = 0.0
        out[..., [3, 40]] = 0.0
        near(plain, query, tables, [n_own] * b, prefix_table, prefix, d**-0.5, out, lse)
