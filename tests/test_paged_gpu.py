"""The paged cache's write and read on the GPU against their definition in 64 bits: codes and scales are
equal, values differ by the roundings of one product and of the output's type."""

from __future__ import annotations

import pytest
import torch

from tests.paged_plain import Cache, quantise_rows

pytestmark = pytest.mark.gpu

# one float32 product, then the output's rounding (half a step each, relative)
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8 + 2.0**-24}


def _tokens(gen: torch.Generator, b: int, t: int, h: int, d: int, dtype: torch.dtype, layout: str) -> tuple[torch.Tensor, torch.Tensor]:
    """keys and values [b, t, h, d] on the GPU in one of several stride patterns."""
    x = torch.randn((b, t, 3, h, d), generator=gen) * torch.rand((b, t, 3, h, 1), generator=gen).exp2()
    x = x.to(dtype).cuda()
    if layout == "packed":
        return x[:, :, 1], x[:, :, 2]
    if layout == "heads first":
        return x[:, :, 1].transpose(1, 2).contiguous().transpose(1, 2), x[:, :, 2].transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "odd":  # rows that no 16-byte load can reach
        flat = torch.zeros((2, b, t, h, d + 3), dtype=dtype, device="cuda")
        flat[0, ..., 1 : d + 1], flat[1, ..., 1 : d + 1] = x[:, :, 1], x[:, :, 2]
        return flat[0, ..., 1 : d + 1], flat[1, ..., 1 : d + 1]
    return x[:, :, 1].contiguous(), x[:, :, 2].contiguous()


@pytest.mark.parametrize("layout", ["plain", "packed", "heads first", "odd"])
@pytest.mark.parametrize("b,t,h,bs", [(1, 1, 1, 16), (3, 5, 2, 16), (2, 40, 3, 32), (5, 1, 8, 128), (1, 131, 5, 64)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("int8,dtype", [(True, torch.bfloat16), (True, torch.float32), (False, torch.bfloat16), (False, torch.float32)])
def test_written_tokens_read_back(int8: bool, dtype: torch.dtype, d: int, b: int, t: int, h: int, bs: int, layout: str) -> None:
    from lazykv_b200 import kernels as K

    gen = torch.Generator().manual_seed(b * 1000 + t * 10 + d)
    keys, values = _tokens(gen, b, t, h, d, dtype, layout)
    starts = [7 * i + (bs - 2 if i == 0 else 0) for i in range(b)]  # the first sequence crosses into its next page at once
    cols = max(-(-(s + t) // bs) for s in starts)
    n_pages = b * cols + 2
    ids = torch.randperm(n_pages, generator=gen)[: b * cols].view(b, cols).to(torch.int32)
    want = Cache(n_pages, h, bs, d, int8, dtype)
    pages, scales = want.pages.cuda(), None if want.scales is None else want.scales.cuda()
    table, first = ids.cuda(), torch.tensor(starts, dtype=torch.int32, device="cuda")
    K.paged_write(keys, values, pages, table, first, scales=scales)
    for i in range(b):
        want.write(ids[i].tolist(), starts[i], keys[i].cpu(), values[i].cpu())
    assert torch.equal(pages.cpu(), want.pages)  # the rows that were not written too
    if int8:
        assert torch.equal(scales.cpu(), want.scales)
    lens = [s + t - (1 if i == 1 else 0) for i, s in enumerate(starts)]  # the second sequence ends a token early
    for out_dtype in ((torch.bfloat16, torch.float32) if int8 else (dtype,)):
        k, v = K.paged_read(pages, table, first, t + 2, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), scales=scales, dtype=out_dtype)
        assert k.shape == (b, t + 2, h, d) and k.dtype == out_dtype and v.dtype == out_dtype
        for i in range(b):
            live = [p for p in range(starts[i], starts[i] + t + 2)]
            wk, wv, _ = want.read(ids[i].tolist(), [p if p < lens[i] else -1 for p in live])
            for got, exact in ((k[i], wk), (v[i], wv)):
                err = (got.double().cpu() - exact).abs()
                assert bool((err <= (HALF[out_dtype] if int8 else 0.0) * exact.abs()).all()), (i, float(err.max()))


def test_codes_at_the_border_of_two_codes() -> None:
    """Quotients next to k + 1/2, where a rounded quotient would choose the wrong side, and exact halves."""
    from lazykv_b200 import kernels as K

    d, n = 128, 512
    gen = torch.Generator().manual_seed(5)
    top = torch.rand((n, 1), generator=gen) * 3 + 0.1
    s = (top.double() / 127).float()
    near = (torch.randint(-126, 126, (n, d), generator=gen).double() + 0.5) * s.double()
    x = near.float()
    x = torch.where(torch.rand((n, d), generator=gen) < 0.3, torch.nextafter(x, torch.full_like(x, torch.inf)), x)
    x = torch.where(torch.rand((n, d), generator=gen) < 0.3, torch.nextafter(x, torch.full_like(x, -torch.inf)), x)
    x[:, 0:1] = top
    x[0] = torch.arange(d) - 63.5  # scale 0.5: exact halves
    x[0, 0] = 63.5
    keys = x.view(1, n, 1, d).cuda()
    pages, scales = torch.zeros((32, 1, 2, 16, d), dtype=torch.int8, device="cuda"), torch.zeros((32, 1, 2, 16), device="cuda")
    table = torch.arange(32, dtype=torch.int32, device="cuda").view(1, 32)
    K.paged_write(keys, -keys, pages, table, torch.zeros(1, dtype=torch.int32, device="cuda"), scales=scales)
    codes, want = quantise_rows(x)
    assert torch.equal(pages[:, 0, 0].reshape(n, d).cpu(), codes) and torch.equal(scales[:, 0, 0].reshape(n).cpu(), want)
    assert torch.equal(pages[:, 0, 1].reshape(n, d).cpu(), -codes)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_zero_tiny_huge_and_non_finite_rows(dtype: torch.dtype) -> None:
    from lazykv_b200 import kernels as K

    d = 64
    x = torch.randn((16, d), generator=torch.Generator().manual_seed(2)).to(dtype)
    x[0] = 0
    x[1] = x[1] * 1e-38  # below the floor of the scale
    x[2] = 0
    x[2, 3] = torch.finfo(dtype).max
    x[2, 4] = -torch.finfo(dtype).max
    x[3, 5] = torch.inf
    x[4, 6] = -torch.inf
    x[5, 7] = torch.nan
    x[6] = torch.nan
    x[7] = -0.0
    keys = x.view(1, 16, 1, d).cuda()
    pages, scales = torch.full((1, 1, 2, 16, d), 5, dtype=torch.int8, device="cuda"), torch.zeros((1, 1, 2, 16), device="cuda")
    table, zero = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    K.paged_write(keys, keys, pages, table, zero, scales=scales)
    codes, want = quantise_rows(x)
    assert torch.equal(pages[0, 0, 0].cpu(), codes)
    assert torch.equal(scales[0, 0, 0].cpu().nan_to_num(-1.0), want.nan_to_num(-1.0))
    back, _ = K.paged_read(pages, table, zero, 16, scales=scales, dtype=torch.float32)
    assert bool(back[0, 3:7].isnan().all()) and bool(back[0, [0, 1, 2, 7, 8]].isfinite().all())


def test_tokens_without_a_page_are_neither_written_nor_read() -> None:
    from lazykv_b200 import kernels as K

    h, bs, d, n_pages = 2, 16, 64, 6
    gen = torch.Generator().manual_seed(9)
    table = torch.tensor([[3, -1, 5], [9, 1, 2**31 - 1], [0, 4, -7], [2, 2, 2]], dtype=torch.int32)  # holes and ids outside [0, 6)
    starts = [10, 14, -3, 45]  # into a hole, from a bad id to a good one, before the start, past the table's end
    keys = torch.randn((4, 20, h, d), generator=gen).bfloat16()
    want = Cache(n_pages, h, bs, d, True)
    pages, scales = want.pages.cuda(), want.scales.cuda()
    first = torch.tensor(starts, dtype=torch.int32, device="cuda")
    wide = torch.full((4, 8), 99, dtype=torch.int32, device="cuda")  # a table that is a view of a wider one
    wide[:, 2:5] = table.cuda()
    K.paged_write(keys.cuda(), keys.cuda(), pages, wide[:, 2:5], first, scales=scales)
    for i in range(4):
        want.write(table[i].tolist(), starts[i], keys[i], keys[i])
    assert torch.equal(pages.cpu(), want.pages) and torch.equal(scales.cpu(), want.scales)
    k, v = K.paged_read(pages, wide[:, 2:5], first, 20, scales=scales, dtype=torch.float32)
    for i in range(4):
        wk, wv, _ = want.read(table[i].tolist(), list(range(starts[i], starts[i] + 20)))
        assert bool(((k[i].cpu().double() - wk).abs() <= 2.0**-24 * wk.abs()).all()) and bool(((v[i].cpu().double() - wv).abs() <= 2.0**-24 * wv.abs()).all())


def test_nothing_to_write_or_read() -> None:
    from lazykv_b200 import kernels as K

    pages = torch.ones((2, 1, 2, 16, 64), dtype=torch.bfloat16, device="cuda")
    none = torch.zeros((0, 1, 1, 64), dtype=torch.bfloat16, device="cuda")
    table, starts = torch.zeros((0, 3), dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    K.paged_write(none, none, pages, table, starts)
    k, _ = K.paged_read(pages, table, starts, 4)
    assert k.shape == (0, 4, 1, 64)
    table, starts = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    k, _ = K.paged_read(pages, table, starts, 0)
    assert k.shape == (1, 0, 1, 64)
    k, v = K.paged_read(pages, table[:, :0], starts, 3)  # a table without columns: no token has a page
    assert float(k.abs().sum() + v.abs().sum()) == 0.0


def test_pages_past_32_bit_offsets() -> None:
    """The last page of a cache whose elements pass 2^31."""
    from lazykv_b200 import kernels as K

    h, bs, d = 64, 128, 128
    n = 2**31 // (h * 2 * bs * d) + 2
    pages = torch.empty((n, h, 2, bs, d), dtype=torch.int8, device="cuda")
    scales = torch.empty((n, h, 2, bs), device="cuda")
    table = torch.tensor([[n - 1]], dtype=torch.int32, device="cuda")
    starts = torch.tensor([5], dtype=torch.int32, device="cuda")
    x = torch.randn((1, 3, h, d), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    K.paged_write(x, -x, pages, table, starts, scales=scales)
    k, v = K.paged_read(pages, table, starts, 3, scales=scales, dtype=torch.float32)
    codes, s = quantise_rows(x.cpu())
    exact = codes.double() * s.double()[..., None]
    assert bool(((k.cpu().double() - exact).abs() <= 2.0**-24 * exact.abs()).all()) and torch.equal(v, -k)
    assert torch.equal(pages[n - 1, :, 0, 5:8].cpu(), codes[0].transpose(0, 1))


def test_out_stream_and_graph() -> None:
    """Into given outputs, on a stream of its own, and replayed from a graph after the inputs changed."""
    from lazykv_b200 import kernels as K

    h, bs, d = 2, 16, 128
    gen = torch.Generator().manual_seed(3)
    pages, scales = torch.zeros((4, h, 2, bs, d), dtype=torch.int8, device="cuda"), torch.zeros((4, h, 2, bs), device="cuda")
    table, starts = torch.tensor([[1, 0], [2, 3]], dtype=torch.int32, device="cuda"), torch.tensor([3, 15], dtype=torch.int32, device="cuda")
    x = torch.randn((2, 4, h, d), generator=gen).bfloat16().cuda()
    out = (torch.empty((2, 4, h, d), dtype=torch.bfloat16, device="cuda"), torch.empty((2, 4, h, d), dtype=torch.bfloat16, device="cuda"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.paged_write(x, x, pages, table, starts, scales=scales)
        got = K.paged_read(pages, table, starts, 4, scales=scales, out=out)
    torch.cuda.current_stream().wait_stream(side)
    assert got[0] is out[0]
    eager = out[0].clone()
    codes, s = quantise_rows(x.cpu())
    exact = codes.double() * s.double()[..., None]
    assert bool(((eager.cpu().double() - exact).abs() <= HALF[torch.bfloat16] * exact.abs()).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.paged_write(x, x, pages, table, starts, scales=scales)
        K.paged_read(pages, table, starts, 4, scales=scales, out=out)
    x.mul_(0.5)  # a power of two: the codes stay, the scales halve
    starts.add_(1)
    graph.replay()
    assert torch.equal(out[0], eager * 0.5)
    assert torch.equal(out[1], out[0])
