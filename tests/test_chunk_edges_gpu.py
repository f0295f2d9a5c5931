"""Chunk attention and attention sums where they can go wrong: missing pages, infinities and NaN in places that a row sees or
does not see, lengths outside the table, scales, strides, streams, graphs, and waits that run out."""

from __future__ import annotations

import math
import time

import pytest
import torch

from tests.test_attention_sums_gpu import check as check_sums
from tests.test_attention_sums_gpu import definition
from tests.test_chunk_attention_gpu import _kernels, _offsets, check
from tests.test_prefix_attention_gpu import build, on_gpu

pytestmark = pytest.mark.gpu


def _i32(x) -> torch.Tensor:  # noqa: ANN001
    return torch.as_tensor(x, dtype=torch.int32, device="cuda")


def _run(cache, query, tables, lens, offsets, prefix_table, prefix, scale, cap=0.0):  # noqa: ANN001, ANN202
    """Both operators on a cache of the CPU, checked against their definitions; returns what they gave."""
    K = _kernels()
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    q, where = query.cuda(), _i32(offsets)
    out, lse = K.chunk_attention(q, pages, table, n, where, scale, scales=scales, prefix_table=ptab, prefix_len=prefix, cap=cap)
    room = len(tables[0]) * cache.bs
    assert K.device_status() == 0
    check(cache, query, tables, lens, offsets, prefix_table, prefix, scale, cap, out, lse)
    got = K.attention_sums(q, lse, pages, table, n, where, scale, cap=cap, scales=scales)
    assert K.device_status() == 0
    check_sums(got, *definition(cache, query, lse.cpu(), tables, lens, offsets, scale, cap, torch.zeros((len(lens), pages.shape[1], room)), None))
    return out, lse, got


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("new", [[3, 40, 1, 0], [70, 1, 30, 1]], ids=["few", "more"])
def test_missing_pages_and_lengths_outside_the_table(int8: bool, new: list[int]) -> None:
    gen = torch.Generator().manual_seed(11)
    lens = [37, 400, 90, 17]
    cache, prefix_table, tables = build(gen, 2, 128, 16, int8, 300, lens)
    prefix_table[2], prefix_table[7], prefix_table[18] = -1, len(cache.pages), 2**31 - 1
    tables[0][1], tables[1][3], tables[1][20] = -5, len(cache.pages) + 3, -1
    tables[2] = [-1] * len(tables[2])
    query = torch.randn((sum(new), 8, 128), generator=gen).bfloat16()
    _run(cache, query, tables, lens, _offsets(new), prefix_table, 300, 128**-0.5)
    _run(cache, query, tables, lens, _offsets(new), prefix_table, 0, 128**-0.5)
    # A length past the table: rows see what the table holds, counted from the length; below zero: nothing.
    _run(cache, query, tables, [37, len(tables[0]) * 16 + 9, 10**6, -4], _offsets(new), prefix_table, 300, 128**-0.5, cap=9.0)


@pytest.mark.parametrize("d", [64, 128])
def test_values_that_are_not_finite(d: int) -> None:
    """In rows of the last page that no token fills, in tokens that some rows of a tile see and others do not, and in
    tokens that all see, in the prefix too."""
    gen = torch.Generator().manual_seed(5)
    new, lens, prefix = [90, 3, 200, 1], [300, 3, 200, 500], 200
    cache, prefix_table, tables = build(gen, 2, d, 16, False, prefix, lens)  # (unused rows hold NaN)
    put = lambda b, pos, j, c, x: cache.pages[tables[b][pos // 16], j, 1, pos % 16].__setitem__(c, x)  # noqa: E731
    put(0, 215, 0, 3, math.inf)      # in the chunk: seen by rows 5 on
    put(0, 215, 0, 9, -math.inf)
    put(0, 250, 0, 3, -math.inf)     # both: NaN from row 40 on
    put(0, 10, 1, 5, math.inf)       # seen by all, in a tile that all see
    put(2, 199, 1, 0, math.nan)      # the last token
    put(2, 0, 1, 1, math.inf)        # the first
    put(3, 499, 0, 2, math.inf)
    cache.pages[prefix_table[12], 0, 1, 7, 4] = math.inf  # token 199 of the prefix: its last tile
    for group in (1, 4):
        query = torch.randn((sum(new), 2 * group, d), generator=gen).bfloat16()
        _run(cache, query, tables, lens, _offsets(new), prefix_table, prefix, d**-0.5)
        _run(cache, query, tables, lens, _offsets(new), prefix_table, 0, d**-0.5, cap=20.0)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_keys_and_scales_that_are_not_finite_reach_only_rows_that_see_them(int8: bool) -> None:
    gen = torch.Generator().manual_seed(6)
    new, lens = [100], [260]
    cache, prefix_table, tables = build(gen, 1, 64, 16, int8, 0, lens)
    for pos, x in ((200, math.nan), (230, math.inf)):
        if int8:
            cache.scales[tables[0][pos // 16], 0, :, pos % 16] = math.nan
        else:
            cache.pages[tables[0][pos // 16], 0, 0, pos % 16, 3] = x
    query = torch.randn((100, 2, 64), generator=gen).bfloat16()
    K = _kernels()
    pages, scales, _, table, n = on_gpu(cache, prefix_table, tables, lens)
    out, lse = K.chunk_attention(query.cuda(), pages, table, n, _i32([0, 100]), 0.125, scales=scales)
    assert not bool(out[:40].isnan().any()) and bool(out[40:].isnan().all())  # row i sees tokens up to 160 + i
    assert not bool(lse[:40].isnan().any()) and bool(lse[40:].isnan().all())
    # (Not to the last bit what they are without the token: a warp's rows take new references together.)
    check(cache, query[:40], tables, [200], [0, 40], prefix_table, 0, 0.125, 0.0, out[:40], lse[:40])
    got = K.attention_sums(query[:40].cuda(), lse[:40], pages, table, _i32([200]), _i32([0, 40]), 0.125, scales=scales)
    assert not bool(got.isnan().any())


@pytest.mark.parametrize("scale", [0.0, -0.3, 40.0, 1e-30])
def test_any_softmax_scale(scale: float) -> None:
    gen = torch.Generator().manual_seed(7)
    new, lens = [50, 140], [200, 300]
    cache, prefix_table, tables = build(gen, 1, 64, 32, False, 70, lens)
    query = torch.randn((190, 2, 64), generator=gen).bfloat16()
    _run(cache, query, tables, lens, _offsets(new), prefix_table, 70, scale)
    _run(cache, query, tables, lens, _offsets(new), prefix_table, 70, scale, cap=7.0)


def test_references_that_are_outgrown() -> None:
    """Scores that rise by hundreds along the tokens: weights have to be taken from new references again and again."""
    gen = torch.Generator().manual_seed(8)
    new, lens = [60, 150], [900, 700]
    cache, prefix_table, tables = build(gen, 1, 64, 16, False, 0, lens)
    for b, n in enumerate(lens):
        for pos in range(n):
            cache.pages[tables[b][pos // 16], 0, 0, pos % 16] *= 1 + pos / 60
    query = (2 * torch.randn((210, 4, 64), generator=gen)).bfloat16()
    _run(cache, query, tables, lens, _offsets(new), prefix_table, 0, 0.125)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_strides_streams_and_two_calls_at_once(int8: bool) -> None:
    K = _kernels()
    gen = torch.Generator().manual_seed(9)
    new, lens = [64, 1, 300], [700, 900, 300]
    cache, prefix_table, tables = build(gen, 2, 64, 16, int8, 150, lens)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    rows, where = sum(new), _i32(_offsets(new))
    base = torch.randn((rows, 12 * 64 + 1), generator=gen).bfloat16().cuda()
    packed = base[:, 1:].unflatten(1, (12, 64))  # unaligned rows of a packed projection
    turned = torch.randn((8, rows, 64), generator=gen).bfloat16().cuda().transpose(0, 1)
    wide = torch.cat([table, torch.full_like(table, 7)], dim=1)[:, : table.shape[1]]  # a table with a row stride

    def call(q, t):  # noqa: ANN001, ANN202
        out, lse = K.chunk_attention(q, pages, t, n, where, 0.125, scales=scales, prefix_table=ptab, prefix_len=150)
        return out, lse, K.attention_sums(q, lse, pages, t, n, where, 0.125, scales=scales)

    want = [call(q.contiguous(), table) for q in (packed[:, 2:10], turned)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for stream, q in zip(streams, (packed[:, 2:10], turned)):
            with torch.cuda.stream(stream):
                got.append(call(q, wide))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert K.device_status() == 0


def test_captured_graphs_follow_lengths_offsets_and_tables() -> None:
    K = _kernels()
    gen = torch.Generator().manual_seed(10)
    cache, prefix_table, tables = build(gen, 2, 128, 16, True, 64, [400, 400, 400])
    pages, scales, ptab, table, _ = on_gpu(cache, prefix_table, tables, [400] * 3)
    rows = 300
    q = torch.randn((rows, 8, 128), generator=gen).bfloat16().cuda()
    lens, where = _i32([1, 1, 1]), _i32([0, 1, 2, 3])
    sums = torch.rand((3, 2, table.shape[1] * 16), generator=gen).cuda()

    def call():  # noqa: ANN202
        out, lse = K.chunk_attention(q, pages, table, lens, where, 0.1, scales=scales, prefix_table=ptab, prefix_len=64)
        return out, lse, K.attention_sums(q, lse, pages, table, lens, where, 0.1, sums=sums, scales=scales)

    call()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(call())
    for n, offsets in (([400, 399, 17], [0, 200, 200, 217]), ([300, 1, 400], [0, 1, 1, 300]), ([0, 0, 0], [0, 0, 0, 0])):
        lens.copy_(_i32(n))
        where.copy_(_i32(offsets))
        live = offsets[-1]
        want = call()
        for graph, out in zip(graphs, outs):
            graph.replay()
            assert torch.equal(out[0][:live], want[0][:live]) and torch.equal(out[1][:live], want[1][:live]) and torch.equal(out[2], want[2])
    assert K.device_status() == 0


@pytest.mark.parametrize("stall", [1, 2], ids=["queries", "weights"])
@pytest.mark.parametrize("new", [[20, 3], [300, 90]], ids=["one row tile", "two row tiles"])
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(int8: bool, new: list[int], stall: int) -> None:
    from lazykv_b200 import _lib

    K = _kernels()
    K.status_attach()
    gen = torch.Generator().manual_seed(12)
    lens = [900, 500]
    cache, prefix_table, tables = build(gen, 2, 64, 16, int8, 100, lens)
    pages, scales, ptab, table, n = on_gpu(cache, prefix_table, tables, lens)
    q, where = torch.randn((sum(new), 4, 64), generator=gen).bfloat16().cuda(), _i32(_offsets(new))

    def call() -> tuple[torch.Tensor, torch.Tensor]:
        done = K.chunk_attention(q, pages, table, n, where, 0.125, scales=scales, prefix_table=ptab, prefix_len=100)
        torch.cuda.synchronize()
        return done

    want = call()
    assert K.device_status(clear=True) == 0
    K.status_poll(clear=True)
    K.debug_set(_lib.LKV_DEBUG_CHUNK_WAIT_NS, 1_000_000)
    K.debug_set(_lib.LKV_DEBUG_CHUNK_STALL_NEXT, stall)
    try:
        began = time.monotonic()
        call()
        took = time.monotonic() - began
    finally:
        K.debug_set(_lib.LKV_DEBUG_CHUNK_STALL_NEXT, 0)
        K.debug_set(_lib.LKV_DEBUG_CHUNK_WAIT_NS, 2_000_000_000)
    with pytest.raises(K.DeviceWaitError):
        K.raise_on_status("test")
    assert K.device_status(clear=True) == _lib.LKV_DEV_WAIT_TIMEOUT
    assert took < 1.0
    again = call()
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    assert K.device_status(clear=True) == 0 and K.status_poll(clear=True) == 0


def test_refusals() -> None:
    K = _kernels()
    pages, table = torch.zeros(4, 2, 2, 16, 64, dtype=torch.bfloat16, device="cuda"), _i32([[0, 1], [2, 3]])
    q, lens, where = torch.zeros(5, 4, 64, dtype=torch.bfloat16, device="cuda"), _i32([5, 9]), _i32([0, 2, 5])
    base = {"query": q, "pages": pages, "table": table, "lens": lens, "offsets": where, "scale": 0.1}
    lse = torch.zeros(5, 4, device="cuda")
    for change in ({"query": q.float()}, {"query": q[:, :3]}, {"query": q[..., :32]}, {"pages": pages.float()}, {"lens": lens[:1]}, {"offsets": where[:2]}, {"cap": -1.0}, {"cap": math.inf},
                   {"table": table.long()}):
        with pytest.raises(ValueError):
            K.chunk_attention(**{**base, **change})
        with pytest.raises(ValueError):
            K.attention_sums(**{**base, **change}, lse=lse)
    for change in ({"prefix_len": 1}, {"prefix_len": 40, "prefix_table": _i32([1, 2])}, {"out": q.float()}, {"lse": lse[:4]}, {"prefix_table": _i32([[1, 2]])}):
        with pytest.raises(ValueError):
            K.chunk_attention(**{**base, **change})
    for change in ({"lse": lse[:4]}, {"last": 0}, {"sums": torch.zeros(2, 2, 30)}, {"sums": torch.zeros(2, 1, 32, device="cuda")}, {"out": torch.zeros(2, 2, 32, dtype=torch.float64, device="cuda")}):
        with pytest.raises(ValueError):
            K.attention_sums(**{**base, "lse": lse, **change})
