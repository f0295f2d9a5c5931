"""take_back() on a tracked batch: the sums are what they would be if only the tokens that stay had come.

Both sides sum the same float32 weights; the row's lse of a call with more tokens may be rounded otherwise. By the bounds of
the operators' own tests an lse is off by less than (d + 4) 2^-24 reach + 2^-21 + n 2^-24 + 4 2^-24 (|lse| + 1), reach <= 30 the largest
sum |q k| scale, n <= 700 keys, |lse| < 30: under 2^-12.5 at d 64, twice that between the two, so a sum moves by less than 2^-11 of
itself. A rejected query's weights are 1 / 300 of the sums and more."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

H, G, D, PAGE = 2, 4, 64, 16


def _batch(quant: str | None):  # noqa: ANN202
    from lazykv_b200.paged import PagedBatch

    return PagedBatch(H, G, D, max_seqs=4, max_tokens=700, n_pages=200, page=PAGE, quant=quant, track=True)


def _near(a, b, ids: list[int]) -> None:  # noqa: ANN001
    for s in ids:
        n = a.lengths[s]
        assert n == b.lengths[s]
        x, y = a.sums[s, :, :n].double(), b.sums[s, :, :n].double()
        assert bool(((x - y).abs() <= 2.0**-11 * y + 2.0**-100).all()), (s, float(((x - y).abs() / y).max()))


def _filled(quant: str | None, gen: torch.Generator):  # noqa: ANN202
    """Two batches alike: a prefix and chunks of three sequences."""
    rand = lambda *s: torch.randn(s, generator=gen).bfloat16().cuda()  # noqa: E731
    a, b = _batch(quant), _batch(quant)
    pk, pv = rand(H, 37, D), rand(H, 37, D)
    ids = [[x.fork() for _ in range(3)] for x in (a, b) if x.set_prefix(pk, pv) is None]
    assert ids[0] == ids[1]
    q, k, v = rand(340, H * G, D), rand(340, H, D), rand(340, H, D)
    for x in (a, b):
        x.chunk(ids[0], [200, 40, 100], q, k, v, 0.125)
    return a, b, ids[0], rand


@pytest.mark.parametrize("quant", ["int8", None])
def test_a_step_with_rejected_drafts(quant: str | None) -> None:
    """Drafts of five tokens, of which each sequence keeps another number, in one go or one by one; then on from there."""
    gen = torch.Generator().manual_seed(1)
    a, b, ids, rand = _filled(quant, gen)
    for turn in range(3):
        q, k, v = rand(3, 5, H * G, D), rand(3, 5, H, D), rand(3, 5, H, D)
        before = a.sums.clone()
        given = q.clone()
        a.step(ids, given, k, v, 0.125)
        given.fill_(9.0)  # the caller's own
        for s, kept in zip(ids, (2, 5, 0)):
            if turn == 1:
                for _ in range(5 - kept):
                    a.take_back(s, 1)
            elif turn == 0:
                a.take_back(s, 5 - kept)
        if turn == 2:
            a.take_back(ids, [3, 0, 5])
        assert torch.equal(a.sums[ids[2]], before[ids[2]])  # nothing of the call stays
        b.step(ids[:1], q[:1, :2], k[:1, :2], v[:1, :2], 0.125)
        b.step(ids[1:2], q[1:2], k[1:2], v[1:2], 0.125)
        _near(a, b, ids)
        with pytest.raises(ValueError, match="tokens to take back"):
            a.take_back(ids[0], 3)  # two of this call's tokens are left: older ones stay
    one = rand(3, 1, H * G, D), rand(3, 1, H, D), rand(3, 1, H, D)
    before = a.sums.clone()
    a.step(ids, *one, 0.125)
    for s in ids:
        a.take_back(s, 1)
    assert torch.equal(a.sums, before)
    for x in (a, b):
        x.step(ids, *one, 0.125)
    _near(a, b, ids)


def test_a_capped_chunk_and_eviction() -> None:
    gen = torch.Generator().manual_seed(2)
    a, b, ids, rand = _filled("int8", gen)
    freq, w = torch.ones(8, device="cuda"), 1 + 0.1 * rand(D)
    q, k, v = rand(100, H * G, D), rand(100, H, D), rand(100, H, D)
    more = {"frequencies": freq, "q_weight": w, "k_weight": w, "cap": 20.0}
    before = a.sums.clone()
    out, lse = a.chunk(ids, [6, 0, 94], q, k, v, 0.125, **more)
    out.zero_(), lse.zero_()
    a.take_back(ids[0], 4)
    with pytest.raises(ValueError, match="all are taken back or none"):
        a.take_back(ids[2], 1)
    assert a.lengths[ids[2]] == 194
    a.take_back(ids[2], 94)
    assert torch.equal(a.sums[ids[2]], before[ids[2]])
    b.chunk(ids[:1], [2], q[:2], k[:2], v[:2], 0.125, **more)
    _near(a, b, ids)
    # In one go, of two calls; a refused one of them leaves them all.
    c = _batch("int8")
    one, two = c.fork(), c.fork()
    c.chunk([one, two], [5, 70], q[:75], k[:75], v[:75], 0.125, **more)
    middle = c.sums.clone()
    c.chunk([two], [3], q[75:78], k[75:78], v[75:78], 0.125, **more)
    for sequences, counts in (([one, two], [1, 4]), ([one, one], [1, 1]), ([one, two], [1]), ([one], [1, 1]), (one, 6)):
        with pytest.raises(ValueError):
            c.take_back(sequences, counts)
    assert c.lengths == {one: 5, two: 73}
    c.take_back([two, one], [3, 2])
    assert c.lengths == {one: 3, two: 70} and torch.equal(c.sums[two], middle[two])
    c.take_back((one,), (3,))
    assert c.lengths[one] == 0 and not bool(c.sums[one].any())
    # What the chunk before did to a sequence without new tokens is still its own to take back.
    a.take_back(ids[1], 5)
    assert a.lengths[ids[1]] == 35
    for x in (a, b):
        x.evict(ids[:1], 64, recent=8)
    assert torch.equal(a.positions[ids[0]], b.positions[ids[0]])  # ranked alike
    with pytest.raises(ValueError):
        a.take_back(ids[0], 1)
    a.drop(ids[0])
    assert a.fork() == ids[0]
    with pytest.raises(ValueError):
        a.take_back(ids[0], 1)


def test_an_untracked_batch_takes_back_any_tokens() -> None:
    from lazykv_b200.paged import PagedBatch

    batch = PagedBatch(H, G, D, max_seqs=2, max_tokens=100, n_pages=20, page=PAGE)
    s, gen = batch.fork(), torch.Generator().manual_seed(3)
    for _ in range(3):
        batch.step([s], *(torch.randn(1, 2, n, D, generator=gen).bfloat16().cuda() for n in (H * G, H, H)), 0.125)
    batch.take_back(s, 5)
    assert batch.lengths[s] == 1


def test_what_is_kept_holds_no_graph() -> None:
    gen = torch.Generator().manual_seed(5)
    a, _, ids, rand = _filled(None, gen)
    for counts in ([3, 3, 3], [3, 80, 0]):
        q = rand(sum(counts), H * G, D).requires_grad_()
        a.chunk(ids, counts, q, rand(sum(counts), H, D), rand(sum(counts), H, D), 0.125)
        call = a._last[ids[0]].call
        assert not (call.query.requires_grad or call.lse.requires_grad or call.sums.requires_grad)
        assert call.query.shape[0] == (9 if counts[1] == 3 else 3)  # the long chunk's rows are not kept
    q = rand(3, 2, H * G, D).requires_grad_()
    a.step(ids, q, rand(3, 2, H, D), rand(3, 2, H, D), 0.125)
    assert not a._last[ids[0]].call.query.requires_grad
    a.take_back(ids, [1, 2, 0])


def test_next_position_counts_what_was_evicted() -> None:
    """What step()'s caller rotates to: the positions that the batch notes, through chunks, evictions and tokens taken back."""
    gen = torch.Generator().manual_seed(4)
    a, _, ids, rand = _filled("int8", gen)
    assert [a.next_position(s) for s in ids] == [37 + 200, 37 + 40, 37 + 100]
    a.evict(ids, 64, recent=8)
    assert [a.lengths[s] for s in ids] == [64, 40, 64]
    want = [37 + 200, 37 + 40, 37 + 100]
    assert [a.next_position(s) for s in ids] == want
    for t, behind in ((3, 0), (1, 3)):
        a.step(ids, rand(3, t, H * G, D), rand(3, t, H, D), rand(3, t, H, D), 0.125)
        for s, first in zip(ids, want):
            n = a.lengths[s]
            assert a.positions[s, :, n - t : n].tolist() == [list(range(first + behind, first + behind + t))] * H
            assert a.next_position(s) == first + behind + t
    a.take_back(ids[0], 1)
    assert a.next_position(ids[0]) == want[0] + 3
