"""Rotated writes against the 64-bit definition: norms, both pairings, partial rotations, ragged and padded chunks, strides,
both types of tokens and of pages."""

from __future__ import annotations

import pytest
import torch

from tests import chunk_plain as P
from tests.paged_plain import quantise_rows

pytestmark = pytest.mark.gpu


def _kernels():  # noqa: ANN202
    from lazykv_b200 import kernels

    return kernels


def _case(dtype: torch.dtype, d: int, h: int, g: int, new: list[int], before: list[int], bs: int, int8: bool, pad: int = 0, seed: int = 0, packed: bool = False):  # noqa: ANN202
    gen = torch.Generator().manual_seed(seed)
    rows, hq = sum(new) + pad, h * g
    if packed:
        qkv = torch.randn(rows, hq + 2 * h, d, generator=gen).to(dtype).cuda()
        q, k, v = qkv[:, :hq], qkv[:, hq : hq + h], qkv[:, hq + h :]
    else:
        q, k, v = (torch.randn(rows, n, d, generator=gen).to(dtype).cuda() for n in (hq, h, h))
    lens = [x + y for x, y in zip(new, before)]
    cols = max(1, max(-(-n // bs) for n in lens))
    n_pages = len(new) * cols + 2
    order = torch.randperm(n_pages, generator=gen).to(torch.int32)
    table = order[: len(new) * cols].reshape(len(new), cols).contiguous()
    pages = torch.full((n_pages, h, 2, bs, d), 77, dtype=torch.int8 if int8 else dtype)
    scales = torch.full((n_pages, h, 2, bs), 5.0) if int8 else None
    offsets = [sum(new[:i]) for i in range(len(new) + 1)]
    return q, k, v, table, pages, scales, lens, offsets


def _i32(x) -> torch.Tensor:  # noqa: ANN001
    return torch.as_tensor(x, dtype=torch.int32).cuda()


# An element is computed with at most 32 roundings of its own pair's size (the sum of d squares 12, the root 3, the
# products with the root and the weight 2, the rotation 3, the cosine and sine and their angle 6) in float32 or float64,
# and rounded once to its type.
def _bound(y: torch.Tensor, size: torch.Tensor, positions: torch.Tensor, dtype: torch.dtype, rounded: bool = True) -> torch.Tensor:
    wide = 2.0**-24 if dtype == torch.bfloat16 else 2.0**-53
    angle = (positions.double().abs() * 2.0**-52)[:, None, None]  # the float64 angle's own rounding, twice
    last = (torch.finfo(dtype).eps / 2 if rounded else 2.0**-24) * y.abs() * (1 + 2.0**-8)
    return last + size * (32 * wide + angle) + torch.finfo(torch.float32).tiny


@pytest.mark.parametrize(("dtype", "d", "h", "g", "new", "before", "bs", "pairs", "interleaved", "norm", "packed"), [
    (torch.bfloat16, 128, 8, 4, [1] * 5, [0, 3, 17, 1000, 31], 16, 64, False, True, True),
    (torch.bfloat16, 128, 2, 7, [3, 0, 70, 1], [0, 5, 61, 15], 32, 16, False, False, False),
    (torch.bfloat16, 64, 4, 1, [129], [0], 64, 32, True, True, False),
    (torch.bfloat16, 64, 1, 3, [0, 0, 1], [9, 0, 0], 16, 12, True, False, True),
    (torch.float32, 128, 2, 2, [5, 9], [100, 0], 128, 64, True, True, False),
    (torch.float32, 64, 3, 5, [2, 33, 1], [7, 16, 0], 16, 12, False, True, True),
    (torch.float32, 64, 8, 1, [700], [3], 32, 0, False, True, False),
])
@pytest.mark.parametrize("int8", [False, True])
def test_against_the_definition(dtype, d, h, g, new, before, bs, pairs, interleaved, norm, packed, int8) -> None:  # noqa: ANN001
    K = _kernels()
    q, k, v, table, pages, scales, lens, offsets = _case(dtype, d, h, g, new, before, bs, int8, pad=2, packed=packed)
    rows = q.shape[0]
    gen = torch.Generator().manual_seed(9)
    positions = torch.randint(-5, 200000, (rows,), generator=gen, dtype=torch.int32)
    freq = (10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(1, pairs))).float()
    qw, kw = ((1 + 0.3 * torch.randn(2, d, generator=gen)).to(dtype).unbind() if norm else (None, None))
    dev_pages, dev_scales = pages.cuda(), None if scales is None else scales.cuda()
    out = torch.full((rows, h * g, d), 7.0, dtype=dtype, device="cuda")
    got = K.paged_write_rotated(q, k, v, positions.cuda(), freq.cuda(), dev_pages, table.cuda(), _i32(lens), _i32(offsets), scales=dev_scales,
                                q_weight=None if qw is None else qw.cuda(), k_weight=None if kw is None else kw.cuda(), eps=1e-5, interleaved=interleaved, out=out)
    assert got is out
    q, k, v = q.cpu(), k.cpu(), v.cpu()
    live = offsets[-1]
    y, size = P.rotate(q, positions, freq, qw, 1e-5, interleaved)
    assert torch.all(out[live:] == 7.0), "rows of no sequence are left as they were"
    err = (out.cpu().double() - y).abs() - _bound(y, size, positions, dtype)
    assert err[:live].max() <= 0
    y, size = P.rotate(k, positions, freq, kw, 1e-5, interleaved)
    bound = _bound(y, size, positions, dtype, rounded=not int8)
    want = pages.clone()
    touched = torch.zeros(pages.shape[:1] + pages.shape[3:4], dtype=torch.bool)
    dev_pages = dev_pages.cpu()
    for r in range(live):
        b, pos = P.place_of(r, offsets, lens)
        page, at = int(table[b, pos // bs]), pos % bs
        touched[page, at] = True
        if int8:
            s = dev_scales[page, :, 0, at].cpu().double()
            top = y[r].abs().amax(-1)
            assert torch.all((s * 127 - top).abs() <= bound[r].amax(-1) + top * 2.0**-23)
            off = (dev_pages[page, :, 0, at].double() * s[:, None] - y[r]).abs()
            # half a step, and what 127 steps of a scale half an ulp off and the value's own error add
            assert torch.all(off <= s[:, None] * (0.5 + 127 * 2.0**-22) + bound[r])
            codes, vs = quantise_rows(v[r])
            assert torch.equal(dev_pages[page, :, 1, at], codes) and torch.equal(dev_scales[page, :, 1, at].cpu(), vs)
        else:
            assert torch.all((dev_pages[page, :, 0, at].double() - y[r]).abs() <= bound[r])
            assert torch.equal(dev_pages[page, :, 1, at], v[r])
    assert torch.equal(dev_pages.transpose(1, 3)[~touched], want.transpose(1, 3)[~touched]), "other rows of the pages stay"


@pytest.mark.parametrize("int8", [False, True])
def test_equal_to_a_plain_write_without_norm_and_rotation(int8: bool) -> None:
    K = _kernels()
    q, k, v, table, pages, scales, lens, offsets = _case(torch.bfloat16, 64, 2, 2, [20], [0], 16, int8)
    k[3, 1, 5], v[4, 0, 6], k[7, 0, 1], v[8] = torch.nan, torch.inf, 3e38, 0.0
    a, b = pages.cuda(), pages.cuda()
    sa, sb = (None, None) if scales is None else (scales.cuda(), scales.cuda())
    none = torch.empty(0, device="cuda")
    out = K.paged_write_rotated(q, k, v, _i32(range(20)), none, a, table.cuda(), _i32(lens), _i32(offsets), scales=sa)
    K.paged_write(k[None], v[None], b, table.cuda(), _i32([0]), scales=sb)
    assert torch.equal(out, q)
    same = {"rtol": 0, "atol": 0, "equal_nan": True}
    torch.testing.assert_close(a, b, **same)
    if int8:
        torch.testing.assert_close(sa, sb, **same)


def test_in_place_unaligned_and_on_another_stream() -> None:
    K = _kernels()
    h, hq, d, rows = 2, 6, 64, 37
    base = torch.randn(rows, (hq + 2 * h) * d + 1).bfloat16().cuda()
    qkv = base[:, 1:].unflatten(1, (hq + 2 * h, d))  # neither the base nor the rows are aligned
    q, k, v = qkv[:, :hq], qkv[:, hq : hq + h], qkv[:, hq + h :]
    pos, freq = _i32(range(rows)), torch.full((32,), 0.25, device="cuda")
    w = (1 + torch.rand(d)).bfloat16().cuda()
    table, lens, offsets = _i32([[1, 0, 2]]), _i32([rows]), _i32([0, rows])
    a, b = torch.zeros((3, h, 2, 16, d), dtype=torch.bfloat16, device="cuda"), torch.zeros((3, h, 2, 16, d), dtype=torch.bfloat16, device="cuda")
    want = K.paged_write_rotated(q.contiguous(), k.contiguous(), v.contiguous(), pos, freq, a, table, lens, offsets, q_weight=w, k_weight=w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = K.paged_write_rotated(q, k, v, pos, freq, b, table, lens, offsets, q_weight=w, k_weight=w, out=q)
    side.synchronize()
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want) and torch.equal(a, b)


def test_missing_pages_long_tables_and_odd_offsets() -> None:
    """Tokens without a page have their query only; offsets that name no rows or rows outside write nothing."""
    K = _kernels()
    h, d = 1, 64
    q, k, v = (torch.randn(8, h, d).bfloat16().cuda() for _ in range(3))
    freq, pos = torch.ones(4, device="cuda"), _i32(range(8))
    pages = torch.zeros((2, h, 2, 16, d), dtype=torch.bfloat16, device="cuda")
    table = _i32([[-1, 1], [7, 0], [0, 1]])
    out = torch.full_like(q, 7.0)
    # sequence 0: rows 1 .. 3 at positions 14 .. 16 (the first page missing), 1: at 15 .. 17 (a bad id, then page 0), 2: before the start
    K.paged_write_rotated(q, k, v, pos, freq, pages, table, _i32([17, 18, 1]), _i32([1, 4, 7, 9]), out=out)
    assert torch.all(out[0] == 7.0) and not torch.any(out[1:] == 7.0)
    y = P.rotate(k.cpu(), pos.cpu(), freq.cpu(), None, 0.0, False)[0]
    got = pages.cpu().double()
    assert (got[1, 0, 0, 0] - y[3, 0]).abs().max() < 0.05 and (got[0, 0, 0, :2] - y[5:7, 0]).abs().max() < 0.05
    assert torch.count_nonzero(got[1, :, :, 1:]) == 0 and torch.count_nonzero(got[0, :, :, 2:]) == 0


def test_refusals() -> None:
    K = _kernels()
    q, k, v, table, pages, _, lens, offsets = _case(torch.bfloat16, 64, 2, 2, [5], [0], 16, False)
    base = {"query": q, "keys": k, "values": v, "positions": _i32(range(5)), "frequencies": torch.ones(8, device="cuda"), "pages": pages.cuda(), "table": table.cuda(),
            "lens": _i32(lens), "offsets": _i32(offsets)}
    for change in ({"query": q[:4]}, {"keys": k[:, :1]}, {"values": v.float()}, {"positions": _i32(range(4))}, {"positions": torch.zeros(5, device="cuda")},
                   {"frequencies": torch.ones(6, device="cuda")}, {"frequencies": torch.ones(36, device="cuda")}, {"lens": _i32([5, 5])}, {"offsets": _i32([0])}, {"eps": -1.0},
                   {"q_weight": torch.ones(64, device="cuda")}, {"k_weight": torch.ones(32, dtype=torch.bfloat16, device="cuda")}, {"out": q[:, :1]},
                   {"keys": k.transpose(1, 2).contiguous().transpose(1, 2)}, {"scales": torch.ones(1, device="cuda")}):
        with pytest.raises(ValueError):
            K.paged_write_rotated(**{**base, **change})
