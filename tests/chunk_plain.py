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


def scores(cache, query: torch.Tensor, b: int, tables: list[list[int]], lens: list[int], offsets: list[int], prefix_table: list[int], prefix: int,  # noqa: ANN001
           scale: float, cap: float):  # noqa: ANN201
    """Of sequence b's chunk, in float64: scores [n, hq, keys] (minus infinity where a row does not see a token; prefix first),
    sum |q k| scale alike (0 there), values [keys, h, d], and the own tokens' mask of pages."""
    n, (_, hq, _) = offsets[b + 1] - offsets[b], query.shape
    h = cache.pages.shape[1]
    own = max(0, min(lens[b], len(tables[b]) * cache.bs))
    kp, vp, okp = cache.read(prefix_table, list(range(prefix)))
    ko, vo, oko = cache.read(tables[b], list(range(own)))
    k, v, there = torch.cat([kp, ko]), torch.cat([vp, vo]), torch.cat([okp, oko])
    q = query[offsets[b] : offsets[b + 1]].double().cpu().view(n, h, hq // h, -1)
    z = torch.einsum("thgd,nhd->thgn", q, k).reshape(n, hq, -1) * scale
    size = torch.einsum("thgd,nhd->thgn", q.abs(), k.abs()).reshape(n, hq, -1) * abs(scale)
    if cap:
        z = cap * torch.tanh(z / cap)
    at = torch.arange(prefix + own) - prefix
    limit = lens[b] - n + 1 + torch.arange(n)
    seen = there & ((at < 0) | (at < limit[:, None]))  # the prefix is in front of every row
    z = torch.where(seen[:, None], z, -torch.inf)
    return z, torch.where(seen[:, None], size, 0.0), v, seen


def attend(cache, query: torch.Tensor, tables: list[list[int]], lens: list[int], offsets: list[int], prefix_table: list[int], prefix: int, scale: float,  # noqa: ANN001
           cap: float):  # noqa: ANN201
    """(out, lse, mass, reach) in float64 of packed queries, as paged_plain.attend has them; NaN rows where a seen value is
    one; infinite values count by their sign whatever their weight."""
    rows, hq, d = query.shape
    h = cache.pages.shape[1]
    out, mass = torch.zeros((rows, hq, d), dtype=torch.float64), torch.zeros((rows, hq, d), dtype=torch.float64)
    lse, reach = torch.full((rows, hq), -math.inf, dtype=torch.float64), torch.zeros((rows, hq), dtype=torch.float64)
    for b in range(len(lens)):
        n, some = offsets[b + 1] - offsets[b], slice(offsets[b], offsets[b + 1])
        if n == 0:
            continue
        z, size, v, seen = scores(cache, query, b, tables, lens, offsets, prefix_table, prefix, scale, cap)
        if z.shape[-1] == 0:
            continue
        lse[some], reach[some] = torch.logsumexp(z, -1), size.amax(-1)
        p = torch.where(torch.isneginf(lse[some])[..., None], 0.0, torch.softmax(z, -1)).view(n, h, hq // h, -1)
        finite = torch.where(v.isfinite(), v, 0.0)
        out[some] = torch.einsum("thgn,nhd->thgd", p, finite).reshape(n, hq, d)
        mass[some] = torch.einsum("thgn,nhd->thgd", p, finite.abs()).reshape(n, hq, d)
        odd = torch.where(v.isfinite(), 0.0, v)
        for c in (~v.isfinite()).flatten(1).any(1).nonzero().flatten().tolist():  # tokens with values that are not finite
            out[some] += torch.where(seen[:, c, None, None, None], odd[c][None, :, None], 0.0).expand(n, h, hq // h, d).reshape(n, hq, d)
    return out, lse, mass, reach
