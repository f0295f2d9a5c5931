"""PagedBatch in chunks and within a budget: the operators together, as a serving loop uses them, and what it refuses."""

from __future__ import annotations

import math

import pytest
import torch

from tests import chunk_plain as P

pytestmark = pytest.mark.gpu

H, G, D, PAGE = 2, 4, 64, 16


def _batch(quant: str | None, **more):  # noqa: ANN003, ANN202
    from lazykv_b200.paged import PagedBatch

    return PagedBatch(H, G, D, max_seqs=4, max_tokens=400, n_pages=90, page=PAGE, quant=quant, **more)


def _rand(gen: torch.Generator):  # noqa: ANN202
    return lambda *s: torch.randn(s, generator=gen).bfloat16().cuda()


def _held(batch, s: int):  # noqa: ANN001, ANN202
    """Keys and values of prefix and own tokens in float64 [h, L, d] each, as the pages hold them."""
    k, v = batch.read(s, dtype=torch.float32 if batch.scales is not None else None)
    return k.double().cpu(), v.double().cpu()


def _attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seen: list[int], scale: float):  # noqa: ANN202
    """(out, weights [h, tokens]) of rows q [n, h * g, d]: row i sees the first seen[i] tokens."""
    z = torch.einsum("thgd,hnd->thgn", q.double().cpu().view(len(seen), H, G, D), k) * scale
    z = z.masked_fill((torch.arange(k.shape[1]) >= torch.tensor(seen)[:, None])[:, None, None], -math.inf)
    p = torch.softmax(z, -1)
    return torch.einsum("thgn,hnd->thgd", p, v).reshape(len(seen), H * G, D), p.sum((0, 2))


@pytest.mark.parametrize("quant", ["int8", None])
def test_a_serving_loop(quant: str | None) -> None:
    """Chunks, steps, evictions and chunks again behind a prefix of odd length; outputs, sums, positions and pages are checked
    against the definition over what the pages hold."""
    gen = torch.Generator().manual_seed(4)
    rand, scale = _rand(gen), D**-0.5
    batch = _batch(quant, track=True)
    batch.set_prefix(rand(H, 37, D), rand(H, 37, D))
    ids = [batch.fork() for _ in range(3)]
    freq = (10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda()
    qw, kw = (1 + 0.2 * rand(D)), (1 + 0.2 * rand(D))
    sums = {s: torch.zeros(H, 0, dtype=torch.float64) for s in ids}
    where = {s: torch.zeros(H, 0, dtype=torch.int64) for s in ids}  # positions of each head's tokens
    nexts = {s: 37 for s in ids}
    for turn, counts in enumerate(([130, 0, 5], [1, 1, 1], None, [40, 200, 1], [1, 1, 1], None, [3, 30, 70])):
        if counts is None:
            before = {s: batch.lengths[s] for s in ids}
            free = len(batch._free_pages)
            batch.evict(ids, 64, recent=10, sinks=2)
            for s in ids:
                n = before[s]
                if n <= 64:
                    continue
                left, ps, pp, moves = P.evict([n], sums[s].float()[None], where[s].int()[None], 64, [nexts[s] - 10], 37 + 2)
                # (the kernel ranks its own float32 sums: the same order but where two weights agree to their last bits)
                got = batch.positions[s, :, :64].long().cpu()
                for j in range(H):
                    assert set(got[j].tolist()) == set(pp[0, j, :64].tolist())
                where[s], sums[s] = got, batch.sums[s, :, :64].double().cpu()
                assert batch.lengths[s] == left[0] == 64 and len(batch._pages_of[s]) == 4
                assert bool((batch.positions[s, :, 64:] == -1).all()) and bool((batch.sums[s, :, 64:] == 0).all())
            assert len(batch._free_pages) > free
            continue
        rows = sum(counts)
        step = counts == [1, 1, 1]
        if step:
            q, k, v = rand(3, 1, H * G, D), rand(3, 1, H, D), rand(3, 1, H, D)
            out, _ = batch.step(ids, q, k, v, scale)
            turned, out = q.view(3, H * G, D).cpu(), out.view(3, H * G, D)
        else:
            q, k, v = rand(rows, H * G, D), rand(rows, H, D), rand(rows, H, D)
            out, _ = batch.chunk(ids, counts, q, k, v, scale, frequencies=freq, q_weight=qw, k_weight=kw)
            pos = torch.cat([torch.arange(nexts[s], nexts[s] + t) for s, t in zip(ids, counts)])
            turned = P.rotate(q.cpu(), pos, freq.cpu(), qw.cpu(), 1e-6, False)[0].bfloat16()
            keys = P.rotate(k.cpu(), pos, freq.cpu(), kw.cpu(), 1e-6, False)[0]
        at = 0
        for s, t in zip(ids, counts):
            if t == 0:
                continue
            kk, vv = _held(batch, s)
            n = kk.shape[1]
            if not step:  # the new keys lie behind the others, turned to the sequence's own positions
                far = (kk[:, n - t :] - keys[at : at + t].transpose(0, 1)).abs().max()
                assert far < (0.05 if quant else 2.0**-7 * 8), float(far)
            want, got = _attend(turned[at : at + t], kk, vv, [n - t + i + 1 for i in range(t)], scale)
            assert (out[at : at + t].double().cpu() - want).abs().max() < 0.03, turn
            where[s] = torch.cat([where[s], torch.arange(nexts[s], nexts[s] + t).expand(H, t)], dim=1)
            sums[s] = torch.cat([sums[s], torch.zeros(H, t, dtype=torch.float64)], dim=1) + got[:, 37:]
            nexts[s] += t
            have = batch.lengths[s]
            assert torch.equal(batch.positions[s, :, :have].long().cpu(), where[s])
            assert (batch.sums[s, :, :have].double().cpu() - sums[s]).abs().max() < 2e-2 * max(1.0, float(sums[s].max())) * 0.05 + 2e-2
            sums[s] = batch.sums[s, :, :have].double().cpu()
            at += t
    from lazykv_b200 import kernels as K

    assert K.device_status() == 0


def test_a_chunk_of_single_tokens_is_a_step() -> None:
    gen = torch.Generator().manual_seed(5)
    rand = _rand(gen)
    a, b = _batch(None, track=True), _batch(None, track=True)
    pk, pv = rand(H, 50, D), rand(H, 50, D)
    for x in (a, b):
        x.set_prefix(pk, pv)
    ia, ib = [a.fork() for _ in range(3)], [b.fork() for _ in range(3)]
    for _ in range(20):
        q, k, v = rand(3, 1, H * G, D), rand(3, 1, H, D), rand(3, 1, H, D)
        one = a.step(ia, q, k, v, 0.125)
        two = b.chunk(ib, [1, 1, 1], q[:, 0], k[:, 0], v[:, 0], 0.125)
        # two roundings of weights to bfloat16 and of the output apart: 2^-8 of sum p |v| and of the output each, |v| < 5
        assert (one[0][:, 0].float() - two[0].float()).abs().max() < 4 * 5 * 2.0**-8
        assert (one[1][:, 0] - two[1]).abs().max() < 1e-4
    assert torch.equal(a.pages[a.table[ia].long()], b.pages[b.table[ib].long()])
    assert (a.sums - b.sums).abs().max() < 1e-4 and torch.equal(a.positions, b.positions)


def test_refused_calls_leave_the_batch_as_it_was() -> None:
    gen = torch.Generator().manual_seed(6)
    rand = _rand(gen)
    batch = _batch("int8", track=True)
    s, t = batch.fork(), batch.fork()
    q, k, v = rand(9, H * G, D), rand(9, H, D), rand(9, H, D)
    batch.chunk([s, t], [4, 5], q, k, v, 0.125)
    state = lambda: (dict(batch.lengths), sorted(batch._free_pages), batch.table.clone(), batch.sums.clone(), batch.positions.clone())  # noqa: E731
    want = state()
    for call in (lambda: batch.chunk([s, s], [4, 5], q, k, v, 0.125), lambda: batch.chunk([s], [4, 5], q, k, v, 0.125), lambda: batch.chunk([s, t], [4, 4], q, k, v, 0.125),
                 lambda: batch.chunk([s, t], [10, -1], q, k, v, 0.125), lambda: batch.chunk([s, t], [4, 5], q, k.float(), v, 0.125),
                 lambda: batch.evict([s, s], 4), lambda: batch.evict([s], 0), lambda: batch.evict([s], 4, recent=3, sinks=2), lambda: batch.take_back(s, 5)):
        with pytest.raises(ValueError):
            call()
        got = state()
        assert got[:2] == want[:2] and all(torch.equal(x, y) for x, y in zip(got[2:], want[2:]))
    with pytest.raises(RuntimeError, match="no room"):
        batch.chunk([s], [397], rand(397, H * G, D), rand(397, H, D), rand(397, H, D), 0.125)
    assert batch.lengths == want[0]
    batch.evict([s, t], 5)  # nothing is longer
    assert batch.lengths == want[0]
    batch.evict([t], 3)
    assert batch.lengths[t] == 3
    with pytest.raises(ValueError):
        batch.take_back(t, 1)  # what is left has moved
    batch.chunk([t], [2], q[:2], k[:2], v[:2], 0.125)
    batch.take_back(t, 2)
    plain = _batch(None)
    with pytest.raises(RuntimeError, match="track"):
        plain.evict([plain.fork()], 3)


def test_nothing_waits_for_the_stream() -> None:
    gen = torch.Generator().manual_seed(7)
    rand = _rand(gen)
    batch = _batch("int8", track=True)
    batch.set_prefix(rand(H, 20, D), rand(H, 20, D))
    ids = [batch.fork() for _ in range(2)]
    q, k, v = rand(60, H * G, D), rand(60, H, D), rand(60, H, D)
    freq = torch.ones(8, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        for _ in range(3):
            batch.chunk(ids, [50, 10], q, k, v, 0.125, frequencies=freq)
            batch.step(ids, q[:2, None], k[:2, None], v[:2, None], 0.125)
            batch.evict(ids, 32, recent=4)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert all(batch.lengths[s] <= 32 for s in ids)
