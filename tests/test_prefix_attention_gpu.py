"""Attention over a shared prefix against its definition in 64 bits.

Bounds, per output element. The kernels round each probability once to bfloat16 before the second
product (half a step: 2^-8 relative), so the sum over keys is off by at most 2^-8 of mass = sum p |v| /
sum p. A score is a float32 sum of d products (two more roundings for the scales): off by at most
delta = (d + 4) 2^-24 reach with reach = max over keys of sum |q k| scale, which moves every weight by a
factor within e^(+-delta), and so do exp2's own error (2^-22) and the float32 sums of n keys (at most
n 2^-24, their worst case): out is off by (2^-8 + 2 (delta + 2^-22 + n 2^-24)) mass, plus half a step of a
bfloat16 output. lse is off by delta + 2^-22 + n 2^-24, plus float32's roundings of its own size.

int8 pages: weights and the scales of values are rounded to f16 instead, relative 2^-11 each (three of them,
with the product of a code and its scale: less than 2^-8), but with a last bit. A reference is set so that the
largest weight times the largest value scale 2^E is 2^7, and f16 steps by 2^-24 at least: a weight times its
scale is off by up to 2^-25 = 2^-32 of that, which a code of 127 makes 2^-32 127 2^E <= 2^-31 vmax (2^E is less
than twice the largest scale, and 127 times that is vmax, the largest magnitude of a value). n keys: at most
n 2^-31 vmax, the sum of the weights being at least the largest. A scale below 2^-14 of 2^E is off by up to
2^-25 of it: weights that sum to one make that 2^-24 vmax."""

from __future__ import annotations

import math

import pytest
import torch

from tests.paged_plain import Cache, attend

pytestmark = pytest.mark.gpu


def build(gen: torch.Generator, h: int, d: int, bs: int, int8: bool, prefix: int, lens: list[int], spare: int = 1, fill: float = math.nan):
    """A cache on the CPU whose pages hold `prefix` shared tokens and each sequence's own; rows that no token
    fills hold NaN (their scales, where the pages are int8), which nothing may read into a result."""
    cols = max([1] + [-(-n // bs) for n in lens])
    pcols = max(1, -(-prefix // bs))
    need = pcols + sum(-(-n // bs) for n in lens)
    cache = Cache(need + spare, h, bs, d, int8, fill=fill)
    order = torch.randperm(need + spare, generator=gen).tolist()
    bias = torch.randn((1, h, d), generator=gen)
    prefix_table, at = order[:pcols], pcols
    kv = lambda n: ((torch.randn((n, h, d), generator=gen) + bias).bfloat16(), torch.randn((n, h, d), generator=gen).bfloat16())  # noqa: E731
    cache.write(prefix_table, 0, *kv(prefix))
    tables = []
    for n in lens:
        own = order[at : at + -(-n // bs)]
        at += len(own)
        cache.write(own, 0, *kv(n))
        tables.append(own + [-1] * (cols - len(own)))
    return cache, prefix_table, tables


def on_gpu(cache: Cache, prefix_table: list[int], tables: list[list[int]], lens: list[int]):
    return (cache.pages.cuda(), None if cache.scales is None else cache.scales.cuda(), torch.tensor(prefix_table, dtype=torch.int32, device="cuda"),
            torch.tensor(tables, dtype=torch.int32, device="cuda").view(len(tables), -1), torch.tensor(lens, dtype=torch.int32, device="cuda"))


def check(cache: Cache, query: torch.Tensor, tables, lens, prefix_table, prefix: int, scale: float, out: torch.Tensor, lse: torch.Tensor) -> None:
    want, wlse, mass, reach = attend(cache, query, tables, lens, prefix_table, prefix, scale)
    d, n = query.shape[-1], prefix + max(lens, default=0)
    delta = (d + 4) * 2.0**-24 * reach
    sums = delta + 2.0**-22 + n * 2.0**-24
    bound = (2.0**-8 + 2 * sums[..., None]) * mass + (2.0**-8 if out.dtype == torch.bfloat16 else 2.0**-23) * want.abs()
    if cache.int8:
        vmax = float((cache.scales[:, :, 1].nan_to_num(0.0) * 127).amax())
        bound = bound + (n * 2.0**-31 + 2.0**-24) * vmax
    err = (out.double().cpu() - want).abs()
    nan, lost = want.isnan(), wlse.isnan()  # where a row attends a NaN it is one
    assert bool(((err <= bound) | nan).all()), (float(err[~nan].max()), float((err / bound.clamp_min(1e-30))[~nan].max()))
    empty = wlse == -math.inf
    got = lse.double().cpu()
    assert torch.equal(out.isnan().cpu(), nan) and torch.equal(got.isnan(), lost)
    assert bool((got[empty] == -math.inf).all()) and bool((out.double().cpu()[empty] == 0).all())
    lerr, lbound = (got - wlse).abs()[~empty & ~lost], (sums + 4 * 2.0**-24 * (wlse.abs() + 1))[~empty & ~lost]
    assert bool((lerr <= lbound).all()), (float(lerr.max()), float(lbound.min()))


CASES = [
    # heads, group, T, page, prefix, own lengths
    (1, 1, 1, 16, 1, [1]),
    (2, 4, 1, 16, 100, [0, 1, 17, 40]),
    (2, 4, 1, 16, 0, [0, 1, 130]),  # no prefix: an empty row
    (1, 1, 5, 32, 33, [0, 3, 5, 6, 70]),  # fewer own tokens than the step's: rows that see none
    (2, 8, 3, 64, 129, [3, 64, 65, 190]),
    (3, 7, 2, 128, 257, [2, 300]),  # 7 query heads a KV head
    (1, 16, 4, 16, 64, [9] * 3),  # 64 rows a sequence: several row tiles
    (2, 2, 1, 16, 1025, [5] * 33),
    (1, 4, 1, 64, 700, [2100, 1, 0]),  # a long own part, split over a cluster
    (2, 1, 1, 16, 3000, [1]),  # one row: the prefix split over many CTAs
    (1, 8, 1, 32, 513, [20 + i for i in range(40)]),  # 320 rows: more than one tile of 256
    (2, 4, 7, 16, 640, [7 + 3 * i for i in range(10)]),  # 280 rows, odd numbers of tokens
    (1, 8, 1, 128, 385, [1] * 50),  # 400 rows: a second block of more than one tile; one token in the last tile
    (1, 4, 1, 64, 384, [3] * 20),  # whole tiles only
    (1, 17, 1, 16, 5000, [2]),  # 17 rows: the fewest that take the tiled prefix; many splits
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "h%d-g%d-t%d-p%d-L%d-b%d" % (c[0], c[1], c[2], c[3], c[4], len(c[5])))
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
def test_matches_the_definition(d: int, int8: bool, case) -> None:  # noqa: ANN001
    from lazykv_b200 import kernels as K

    h, g, t, bs, prefix, lens = case
    gen = torch.Generator().manual_seed(sum(lens) + prefix + d)
    cache, prefix_table, tables = build(gen, h, d, bs, int8, prefix, lens)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    query = (1.5 * torch.randn((len(lens), t, h * g, d), generator=gen)).bfloat16()
    for dtype in (torch.float32, torch.bfloat16):
        out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, prefix, d**-0.5, scales=scales, out_dtype=dtype)
        assert out.dtype == dtype
        check(cache, query, tables, lens, prefix_table, prefix, d**-0.5, out, lse)
    assert K.device_status() == 0


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("b", [2, 40])
def test_missing_pages_are_not_attended(b: int, int8: bool) -> None:
    """Holes and ids outside the cache, in the prefix and in the sequences' own tables; lengths past the table."""
    from lazykv_b200 import kernels as K

    h, g, d, bs, prefix = 2, 4, 128, 16, 400
    lens = [37 + i for i in range(b)]
    gen = torch.Generator().manual_seed(6)
    cache, prefix_table, tables = build(gen, h, d, bs, int8, prefix, lens)
    prefix_table[2], prefix_table[7], prefix_table[24] = -1, len(cache.pages), 2**31 - 1
    tables[0][1], tables[1] = -5, [-1] * len(tables[1])
    if b > 2:
        tables[2][0] = len(cache.pages) + 3
        lens[3], lens[4] = 10**6, -9  # longer than its table, negative
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    query = torch.randn((b, 1, h * g, d), generator=gen).bfloat16()
    out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, prefix, d**-0.5, scales=scales, out_dtype=torch.float32)
    room = len(tables[0]) * bs
    # A length past the table reaches its end, and holes there (-1) have no tokens.
    check(cache, query, tables, [min(x, room) for x in lens], prefix_table, prefix, d**-0.5, out, lse)


@pytest.mark.parametrize("b", [2, 40])
def test_a_prefix_with_no_page_at_all(b: int) -> None:
    from lazykv_b200 import kernels as K

    gen = torch.Generator().manual_seed(16)
    lens = [0 if i % 2 else 5 for i in range(b)]
    cache, prefix_table, tables = build(gen, 1, 64, 16, False, 300, lens)
    prefix_table = [-1] * len(prefix_table)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    query = torch.randn((b, 1, 4, 64), generator=gen).bfloat16()
    out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, 300, 0.125, out_dtype=torch.float32)
    check(cache, query, tables, lens, prefix_table, 300, 0.125, out, lse)
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_values_that_a_row_does_not_see_never_reach_it(int8: bool) -> None:
    """The last drafted token's key and value are not finite: only the query that sees it is affected."""
    from lazykv_b200 import kernels as K

    h, g, d, bs, t = 1, 4, 128, 16, 4
    lens = [30, 4]
    gen = torch.Generator().manual_seed(8)
    cache, prefix_table, tables = build(gen, h, d, bs, int8, 50, lens)
    for i, bad in ((0, torch.inf), (1, torch.nan)):
        x = torch.randn((1, h, d), generator=gen).bfloat16()
        x[..., 5] = bad
        cache.write(tables[i], lens[i] - 1, x, x)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    query = torch.randn((2, t, h * g, d), generator=gen).bfloat16()
    out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, 50, d**-0.5, scales=scales, out_dtype=torch.float32)
    assert bool(out[:, : t - 1].isfinite().all())
    # the rows before the last one: as with that token taken away
    less = [x - 1 for x in lens]
    cut = K.prefix_attention(query[:, : t - 1].contiguous().cuda(), pages, table, torch.tensor(less, dtype=torch.int32, device="cuda"), ptab, 50, d**-0.5,
                             scales=scales, out_dtype=torch.float32)
    want, wlse, mass, _ = attend(cache, query[:, : t - 1], tables, less, prefix_table, 50, d**-0.5)
    for got in (out[:, : t - 1], cut[0]):
        assert bool(((got.double().cpu() - want).abs() <= 2.0**-7 * mass).all())
    assert bool(((lse[:, : t - 1].double().cpu() - wlse).abs() <= 1e-3).all())
    assert bool(out[:, t - 1].isnan().any())


def test_a_query_of_nan_gives_nan_and_leaves_the_others() -> None:
    from lazykv_b200 import kernels as K

    for b in (3, 40):
        gen = torch.Generator().manual_seed(18)
        lens = [6] * b
        cache, prefix_table, tables = build(gen, 1, 64, 16, False, 200, lens)
        pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
        query = torch.randn((b, 1, 4, 64), generator=gen).bfloat16()
        query[1, 0, 2] = torch.nan
        out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, 200, 0.125, out_dtype=torch.float32)
        hit = torch.zeros((b, 1, 4), dtype=torch.bool)
        hit[1, 0, 2] = True
        assert bool(out.cpu()[hit].isnan().all()) and bool(lse.cpu()[hit].isnan().all()) and bool(out.cpu()[~hit].isfinite().all())


@pytest.mark.parametrize("spread", [1e-3, 30.0])
@pytest.mark.parametrize("b", [1, 40])
def test_flat_and_peaked_scores(b: int, spread: float) -> None:
    """Nearly equal weights, and scores of hundreds, where the running maximum moves often."""
    from lazykv_b200 import kernels as K

    h, g, d = 1, 4, 64
    lens = [11] * b
    gen = torch.Generator().manual_seed(19)
    cache, prefix_table, tables = build(gen, h, d, 16, False, 900, lens)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    query = (spread * torch.randn((b, 1, h * g, d), generator=gen)).bfloat16()
    out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, 900, d**-0.5, out_dtype=torch.float32)
    check(cache, query, tables, lens, prefix_table, 900, d**-0.5, out, lse)


@pytest.mark.parametrize("b", [3, 40])
def test_strides_streams_given_outputs_and_graphs(b: int) -> None:
    """Query slices of a packed projection, misaligned queries, two streams at once, and a captured step
    whose lengths and tables change between replays, beside another captured step."""
    from lazykv_b200 import kernels as K

    h, g, d, bs = 2, 4, 64, 16
    lens = [5 + i for i in range(b)]
    gen = torch.Generator().manual_seed(21)
    cache, prefix_table, tables = build(gen, h, d, bs, True, 500, lens)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    packed = torch.randn((b, 1, h * g + 2 * h, d), generator=gen).bfloat16().cuda()
    q = packed[:, :, : h * g]
    base, base_lse = K.prefix_attention(q.contiguous(), pages, table, n, ptab, 500, 0.125, scales=scales)
    out, lse = K.prefix_attention(q, pages, table, n, ptab, 500, 0.125, scales=scales)
    assert torch.equal(out, base) and torch.equal(lse, base_lse)
    flat = torch.zeros(b * h * g * d + 1, dtype=torch.bfloat16, device="cuda")
    flat[1:] = q.reshape(-1)
    out, lse = K.prefix_attention(flat[1:].view(b, 1, h * g, d), pages, table, n, ptab, 500, 0.125, scales=scales)
    assert torch.equal(out, base) and torch.equal(lse, base_lse)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                got.append(K.prefix_attention(q, pages, table, n, ptab, 500, 0.125, scales=scales))
    torch.cuda.synchronize()
    assert all(torch.equal(a, base) and torch.equal(c, base_lse) for a, c in got)
    graphs, outs = [], []
    for _ in range(2):
        o, l = torch.empty_like(base), torch.empty_like(base_lse)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            K.prefix_attention(q, pages, table, n, ptab, 500, 0.125, scales=scales, out=o, lse=l)
        graphs.append(graph)
        outs.append((o, l))
    n.sub_(3)
    table[0].fill_(-1)
    ptab[3] = -1
    again, again_lse = K.prefix_attention(q, pages, table, n, ptab, 500, 0.125, scales=scales)
    assert not torch.equal(again, base)
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for o, l in outs:
        assert torch.equal(o, again) and torch.equal(l, again_lse)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("b", [3, 40])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.5])
def test_any_softmax_scale(scale: float, b: int, int8: bool) -> None:
    from lazykv_b200 import kernels as K

    gen = torch.Generator().manual_seed(31)
    lens = [9 + i % 5 for i in range(b)]
    cache, prefix_table, tables = build(gen, 1, 64, 16, int8, 200, lens)
    prefix_table[3] = -1  # missing pages and a last tile that is not full, under a scale of zero too
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    query = torch.randn((b, 1, 4, 64), generator=gen).bfloat16()
    out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, 200, scale, scales=scales, out_dtype=torch.float32)
    check(cache, query, tables, lens, prefix_table, 200, scale, out, lse)


@pytest.mark.parametrize("b", [3, 40])
@pytest.mark.parametrize("up", [-60, 0, 60])
def test_int8_pages_of_any_magnitude(b: int, up: int) -> None:
    """Queries times 2^up under a softmax scale of 2^-up, values times 2^up or 2^-up: powers of two change no
    rounding of float32, and those of the f16 operands are taken from them."""
    from lazykv_b200 import kernels as K

    gen = torch.Generator().manual_seed(32)
    lens = [9 + i % 5 for i in range(b)]
    cache, prefix_table, tables = build(gen, 1, 64, 16, True, 200, lens, fill=0.0)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    query = torch.randn((b, 1, 4, 64), generator=gen).bfloat16()
    base = K.prefix_attention(query.cuda(), pages, table, n, ptab, 200, 0.125, scales=scales, out_dtype=torch.float32)
    big = (query.float() * 2.0**up).bfloat16().cuda()
    out, lse = K.prefix_attention(big, pages, table, n, ptab, 200, 0.125 * 2.0**-up, scales=scales, out_dtype=torch.float32)
    assert torch.equal(out, base[0]) and torch.equal(lse, base[1])
    scales[:, :, 1] *= 2.0**up  # the references move with the values: their sums are rounded at other places
    out, lse = K.prefix_attention(query.cuda(), pages, table, n, ptab, 200, 0.125, scales=scales, out_dtype=torch.float32)
    assert bool(((out * 2.0**-up - base[0]).abs() <= 2.0**-10 * base[0].abs().amax()).all())
    # lse is a difference of two numbers of up to 70: their float32 roundings
    assert bool(((lse - base[1]).abs() <= 6 * 70 * 2.0**-24).all())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,t", [(2, 1), (3, 4), (40, 1)])
def test_scales_of_unseen_rows_do_not_count(b: int, t: int, d: int) -> None:
    """int8 pages whose rows past the lists' ends hold scales that are numbers, huge ones: the same bits as with NaN."""
    from lazykv_b200 import kernels as K

    got = []
    for fill in (math.nan, 1e30):
        gen = torch.Generator().manual_seed(b)
        lens = [5 + 7 * i for i in range(b)]
        cache, prefix_table, tables = build(gen, 2, d, 16, True, 203, lens, fill=fill)
        pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
        q = torch.randn((b, t, 2, d), generator=gen).bfloat16().cuda()
        got.append(K.prefix_attention(q, pages, table, n, ptab, 203, d**-0.5, scales=scales, out_dtype=torch.float32))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b", [1, 40])
def test_a_drafted_token_counts_for_no_row_before_it(b: int, d: int) -> None:
    """int8: the step's last token has values 2^40 times the others'; the rows before it keep the others' bound."""
    from lazykv_b200 import kernels as K

    gen = torch.Generator().manual_seed(d)
    t, lens = 3, [3 + i for i in range(b)]
    cache, prefix_table, tables = build(gen, 2, d, 16, True, 90, lens)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    ordinary = float((cache.scales[:, :, 1].nan_to_num(0.0) * 127).amax())
    for i, m in enumerate(lens):
        page = tables[i][(m - 1) // 16]
        scales[page, :, 1, (m - 1) % 16] *= 2.0**40
        cache.scales[page, :, 1, (m - 1) % 16] *= 2.0**40
    query = torch.randn((b, t, 4, d), generator=gen).bfloat16()
    out, _ = K.prefix_attention(query.cuda(), pages, table, n, ptab, 90, d**-0.5, scales=scales, out_dtype=torch.float32)
    want, _, mass, reach = attend(cache, query, tables, lens, prefix_table, 90, d**-0.5)
    keys = 90 + max(lens)
    sums = (d + 4) * 2.0**-24 * reach + 2.0**-22 + keys * 2.0**-24
    bound = (2.0**-8 + 2 * sums[..., None]) * mass + 2.0**-23 * want.abs() + (keys * 2.0**-31 + 2.0**-24) * ordinary
    err = (out.double().cpu() - want).abs()[:, : t - 1]
    assert bool((err <= bound[:, : t - 1]).all()), float((err / bound[:, : t - 1]).max())


def test_one_result_for_one_input() -> None:
    """The same call gives the same bits every time (no atomics order its sums)."""
    from lazykv_b200 import kernels as K

    for b, h, g, prefix in ((4, 2, 4, 3000), (64, 2, 4, 2000)):
        gen = torch.Generator().manual_seed(b)
        lens = [100] * b
        cache, prefix_table, tables = build(gen, h, 64, 16, False, prefix, lens)
        pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
        q = torch.randn((b, 1, h * g, 64), generator=gen).bfloat16().cuda()
        first = K.prefix_attention(q, pages, table, n, ptab, prefix, 0.125)
        for _ in range(10):
            out, lse = K.prefix_attention(q, pages, table, n, ptab, prefix, 0.125)
            assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


def test_an_empty_batch() -> None:
    from lazykv_b200 import kernels as K

    pages = torch.zeros((1, 1, 2, 16, 64), dtype=torch.bfloat16, device="cuda")
    out, lse = K.prefix_attention(torch.zeros((0, 1, 4, 64), dtype=torch.bfloat16, device="cuda"), pages, torch.zeros((0, 1), dtype=torch.int32, device="cuda"),
                                  torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), 5, 0.125)
    assert out.shape == (0, 1, 4, 64) and lse.shape == (0, 1, 4)
