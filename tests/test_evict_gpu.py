"""Eviction against its definition: which tokens stay, where they go, ties, protected tokens, odd sums, one CTA and clusters."""

from __future__ import annotations

import pytest
import torch

from tests import chunk_plain as P

pytestmark = pytest.mark.gpu


def _kernels():  # noqa: ANN202
    from lazykv_b200 import kernels

    return kernels


def _i32(x) -> torch.Tensor:  # noqa: ANN001
    return torch.as_tensor(x, dtype=torch.int32)


def _cache(batch: int, h: int, cap: int, bs: int, d: int, kind: str, seed: int):  # noqa: ANN202
    gen = torch.Generator().manual_seed(seed)
    cols = -(-cap // bs)
    n_pages = batch * cols + 1
    table = torch.randperm(n_pages, generator=gen).to(torch.int32)[: batch * cols].reshape(batch, cols).contiguous()
    if kind == "int8":
        return table, torch.randint(-127, 128, (n_pages, h, 2, bs, d), generator=gen, dtype=torch.int8), torch.rand((n_pages, h, 2, bs), generator=gen)
    return table, torch.randn((n_pages, h, 2, bs, d), generator=gen).to(torch.bfloat16 if kind == "bf16" else torch.float32), None


def _moved(x: torch.Tensor, table: torch.Tensor, moves, bs: int) -> torch.Tensor:  # noqa: ANN001
    y = x.clone()
    for b, heads in enumerate(moves):
        for j, pairs in enumerate(heads):
            for of, to in pairs:
                src, dst = int(table[b, of // bs]), int(table[b, to // bs])
                if 0 <= src < x.shape[0] and 0 <= dst < x.shape[0]:
                    y[dst, j, :, to % bs] = x[src, j, :, of % bs]
    return y


@pytest.mark.parametrize(("batch", "h", "lens", "cap", "keep", "bs", "d", "kind", "in_place"), [
    (1, 1, [5], 16, 3, 16, 64, "bf16", False),
    (3, 2, [1, 40, 64], 64, 24, 16, 128, "int8", True),
    (4, 8, [130, 0, 33, 129], 144, 128, 16, 128, "bf16", True),
    (2, 3, [5000, 1777], 5008, 1000, 16, 64, "int8", False),   # two CTAs and more a head
    (1, 2, [40000], 40000, 39000, 64, 64, "bf16", False),      # a cluster of eight, few tokens dropped
    (1, 1, [140001], 140032, 70, 128, 64, "f32", True),        # slices longer than shared memory holds
    (2, 160, [300, 299], 320, 100, 32, 128, "f32", False),     # more heads than SMs
])
def test_against_the_definition(batch, h, lens, cap, keep, bs, d, kind, in_place) -> None:  # noqa: ANN001
    K = _kernels()
    table, pages, scales = _cache(batch, h, cap, bs, d, kind, seed=cap + keep)
    gen = torch.Generator().manual_seed(1)
    sums = torch.exp(2 * torch.randn((batch, h, cap), generator=gen)) * (torch.rand((batch, h, cap), generator=gen) > 0.3)
    positions = torch.randperm(cap * h, generator=gen).to(torch.int32)[:cap].expand(batch, h, cap).contiguous()
    since = [cap * h - 40] * batch
    want_len, want_s, want_p, moves = P.evict(lens, sums, positions, keep, since, 3)
    ds, dp, dpages, dscales = sums.cuda(), positions.cuda(), pages.cuda(), None if scales is None else scales.cuda()
    left, got_s, got_p = K.paged_evict(dpages, table.cuda(), _i32(lens).cuda(), ds, dp, keep, since=_i32(since).cuda(), sinks=3, scales=dscales,
                                       out=(ds, dp) if in_place else None)
    assert left.tolist() == want_len
    assert torch.equal(got_p.cpu(), want_p)
    assert torch.equal(got_s.cpu(), want_s)
    assert torch.equal(dpages.cpu(), _moved(pages, table, moves, bs))
    if scales is not None:
        assert torch.equal(dscales.cpu(), _moved(scales, table, moves, bs))
    if not in_place:
        assert torch.equal(ds.cpu(), sums) and torch.equal(dp.cpu(), positions)


def test_ties_protected_tokens_and_odd_sums() -> None:
    K = _kernels()
    table, pages, _ = _cache(5, 1, 64, 16, 64, "bf16", seed=3)
    sums = torch.zeros(5, 1, 64)
    sums[1] = torch.arange(64.0)
    sums[2, 0, ::3], sums[2, 0, 1::3] = torch.nan, torch.inf
    sums[3, 0, :32], sums[3, 0, 32:] = -0.0, 0.0
    sums[4] = -torch.rand(64) * torch.tensor([1e-45, 1e38]).repeat(32)
    sums[4, 0, 7] = -torch.inf
    positions = torch.arange(64, dtype=torch.int32).expand(5, 1, 64).contiguous()
    lens, since = [64] * 5, [64, 20, 64, 64, 50]  # sequence 1 protects more than are kept
    want_len, want_s, want_p, moves = P.evict(lens, sums, positions, 30, since, 2)
    dpages = pages.cuda()
    left, got_s, got_p = K.paged_evict(dpages, table.cuda(), _i32(lens).cuda(), sums.cuda(), positions.cuda(), 30, since=_i32(since).cuda(), sinks=2)
    assert left.tolist() == want_len and torch.equal(got_p.cpu(), want_p)
    assert torch.equal(got_s.cpu().view(torch.int32), want_s.view(torch.int32))
    assert torch.equal(dpages.cpu(), _moved(pages, table, moves, 16))


def test_missing_pages_and_lengths_outside() -> None:
    """A token without a page is ranked and not moved; lengths below zero and past the slots count as those."""
    K = _kernels()
    table, pages, _ = _cache(3, 2, 48, 16, 64, "bf16", seed=4)
    table[0, 2], table[1, 0] = -1, 99
    gen = torch.Generator().manual_seed(2)
    sums = torch.rand((3, 2, 48), generator=gen)
    positions = torch.arange(48, dtype=torch.int32).expand(3, 2, 48).contiguous()
    lens = [48, 1000, -7]
    want_len, want_s, want_p, moves = P.evict(lens, sums, positions, 20, None, 0)
    dpages = pages.cuda()
    left, got_s, got_p = K.paged_evict(dpages, table.cuda(), _i32(lens).cuda(), sums.cuda(), positions.cuda(), 20)
    assert left.tolist() == want_len and torch.equal(got_p.cpu(), want_p) and torch.equal(got_s.cpu(), want_s)
    assert torch.equal(dpages.cpu(), _moved(pages, table, moves, 16))


def test_captured_and_replayed_with_other_lengths() -> None:
    K = _kernels()
    table, pages, _ = _cache(2, 4, 256, 16, 64, "bf16", seed=6)
    gen = torch.Generator().manual_seed(3)
    sums = torch.rand((2, 4, 256), generator=gen)
    positions = torch.arange(256, dtype=torch.int32).expand(2, 4, 256).contiguous()
    dpages, dlens, ds, dp, dt = pages.cuda(), _i32([3, 3]).cuda(), sums.cuda(), positions.cuda(), table.cuda()
    K.paged_evict(dpages, dt, dlens, ds, dp, 100)  # (three tokens: nothing moves)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        left, got_s, got_p = K.paged_evict(dpages, dt, dlens, ds, dp, 100)
    for lens in ([256, 101], [99, 200]):
        dpages.copy_(pages)
        dlens.copy_(_i32(lens))
        graph.replay()
        want_len, want_s, want_p, moves = P.evict(lens, sums, positions, 100, None, 0)
        assert left.tolist() == want_len and torch.equal(got_p.cpu(), want_p) and torch.equal(got_s.cpu(), want_s)
        assert torch.equal(dpages.cpu(), _moved(pages, table, moves, 16))


def test_refusals() -> None:
    K = _kernels()
    table, pages, _ = _cache(2, 1, 32, 16, 64, "bf16", seed=7)
    lens, sums, positions = _i32([32, 32]).cuda(), torch.zeros(2, 1, 32, device="cuda"), torch.zeros(2, 1, 32, dtype=torch.int32, device="cuda")
    pages, table = pages.cuda(), table.cuda()
    for change in ({"keep": 0}, {"keep": 2**31}, {"sinks": -1}, {"sums": sums[:, :, ::2]}, {"sums": sums.double()}, {"positions": positions.long()}, {"lens": lens[:1]},
                   {"since": lens[:1]}, {"out": (sums[:1], positions)}, {"pages": pages[0]}, {"scales": sums}):
        args = {"pages": pages, "table": table, "lens": lens, "sums": sums, "positions": positions, "keep": 4, **change}
        with pytest.raises(ValueError):
            K.paged_evict(**args)
