"""Plain 64-bit forms of the packed-chunk operators (rotated write, chunk attention, attention sums, eviction), from
their definitions, token by token where that is clearest. Test infrastructure only."""

from __future__ import annotations

import math

import torch


def place_of(row: int, offsets: list[int], lens: list[int]) -> tuple[int, int] | None:
    """(sequence, position in its cache) of a packed row, or None where it belongs to no sequence."""
    for b in range(len(lens)):
        if offsets[b] <= row < offsets[b + 1]:
            return b, lens[b] - offsets[b + 1] + row
    return None


def rotate(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, weight: torch.Tensor | None, eps: float,
           interleaved: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, size) in float64 of rows x [rows, heads, d]: size is |a| + |b| of an element's normalised pair, from which a test
    derives its bound."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    n = frequencies.numel()
    a = list(range(0, 2 * n, 2)) if interleaved else list(range(n))
    b = list(range(1, 2 * n, 2)) if interleaved else list(range(n, 2 * n))
    t = (positions.double()[:, None] * frequencies.double())[:, None]
    out, size = y.clone(), y.abs()
    out[..., a], out[..., b] = y[..., a] * t.cos() - y[..., b] * t.sin(), y[..., b] * t.cos() + y[..., a] * t.sin()
    size[..., a] = size[..., b] = y[..., a].abs() + y[..., b].abs()
    return out, size


def evict(lens: list[int], sums: torch.Tensor, positions: torch.Tensor, keep: int, since: list[int] | None, sinks: int):  # noqa: ANN201
    """(lens left, sums, positions, moves): moves[b][j] lists (from, to) slots."""
    batch, h, cap = sums.shape
    left, out_s, out_p = [], torch.zeros_like(sums), torch.full_like(positions, -1)
    moves = [[[] for _ in range(h)] for _ in range(batch)]
    for b in range(batch):
        n = max(0, min(lens[b], cap))
        left.append(min(n, keep))
        for j in range(h):
            s, p = sums[b, j].tolist(), positions[b, j].tolist()
            safe = [p[i] < sinks or (since is not None and p[i] >= since[b]) for i in range(n)]
            rank = sorted(range(n), key=lambda i: (not safe[i], 0 if safe[i] else math.inf if math.isnan(s[i]) else -s[i], i))
            # NaN sorts behind minus infinity: both have the key inf; a NaN comes after every number
            numbers = [i for i in rank if safe[i] or not math.isnan(s[i])]
            kept = set((numbers + [i for i in rank if not safe[i] and math.isnan(s[i])])[:keep])
            slots = list(range(left[b]))
            late = sorted(i for i in kept if i >= left[b])
            for to, of in zip([i for i in slots if i not in kept], late):
                slots[to] = of
                moves[b][j].append((of, to))
            for i, of in enumerate(slots):
                out_s[b, j, i], out_p[b, j, i] = sums[b, j, of], positions[b, j, of]
    return left, out_s, out_p, moves
