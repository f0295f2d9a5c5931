"""Plain 64-bit forms of the paged cache, the shared-prefix attention and draft verification, from their
definitions, one row at a time where that is clearest. Test infrastructure only."""

from __future__ import annotations

import math

import torch

FLT_MIN = 2.0**-126
SCALE_MAX = float.fromhex("0x1.020406p+121")  # the largest float32 whose 127-fold is one too


def quantise_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes int8, scales float32) of x [..., d]: s = max(max |x| / 127, FLT_MIN) in float32 (SCALE_MAX at most), code the whole
    number nearest to x / s (halfway: even; the quotient in 64 bits); rows with an infinity or NaN: s = NaN, codes 0."""
    xd = x.double()
    top = xd.abs().amax(-1)
    bad = ~torch.isfinite(xd).all(-1)
    s = (torch.where(bad, 0.0, top) / 127.0).float().clamp(FLT_MIN, SCALE_MAX)
    codes = torch.round(torch.where(bad[..., None], 0.0, xd) / s.double()[..., None]).to(torch.int8)
    return codes, torch.where(bad, torch.nan, s)


class Cache:
    """Pages of h heads with shuffled page ids, filled token by token on the CPU."""

    def __init__(self, n_pages: int, h: int, bs: int, d: int, int8: bool, dtype: torch.dtype = torch.bfloat16, fill: float = 0.0) -> None:
        self.bs, self.int8 = bs, int8
        self.pages = torch.full((n_pages, h, 2, bs, d), 77 if int8 else fill, dtype=torch.int8 if int8 else dtype)
        self.scales = torch.full((n_pages, h, 2, bs), fill) if int8 else None

    def write(self, table: list[int], start: int, keys: torch.Tensor, values: torch.Tensor) -> None:
        """keys / values [T, h, d] to positions start ..; tokens without a page are dropped."""
        for t in range(keys.shape[0]):
            pos = start + t
            if pos < 0 or pos // self.bs >= len(table):
                continue
            page = table[pos // self.bs]
            if not 0 <= page < self.pages.shape[0]:
                continue
            for kv, x in enumerate((keys[t], values[t])):
                if self.int8:
                    self.pages[page, :, kv, pos % self.bs], self.scales[page, :, kv, pos % self.bs] = quantise_rows(x)
                else:
                    self.pages[page, :, kv, pos % self.bs] = x

    def read(self, table: list[int], positions: list[int]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """(keys, values) [n, h, d] in float64 (zeros where a token has no page), and which have one."""
        h, d = self.pages.shape[1], self.pages.shape[4]
        out = torch.zeros((2, len(positions), h, d), dtype=torch.float64)
        there = torch.zeros(len(positions), dtype=torch.bool)
        for i, pos in enumerate(positions):
            if pos < 0 or pos // self.bs >= len(table) or not 0 <= table[pos // self.bs] < self.pages.shape[0]:
                continue
            page, there[i] = table[pos // self.bs], True
            x = self.pages[page, :, :, pos % self.bs].double()  # [h, 2, d]
            if self.int8:
                x = x * self.scales[page, :, :, pos % self.bs].double()[..., None]
            out[:, i] = x.transpose(0, 1)
        return out[0], out[1], there


def attend(cache: Cache, query: torch.Tensor, tables: list[list[int]], lens: list[int], prefix_table: list[int], prefix_len: int,
           scale: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(out, lse, mass, reach) in float64 of query [B, T, hq, d] (bfloat16): mass is sum p |v| / sum p per
    output element and reach the largest sum |q k| scale of a row, from which a test derives its bounds."""
    b, t, hq, d = query.shape
    h = cache.pages.shape[1]
    g = hq // h
    q = query.double().cpu()
    out, mass = torch.zeros((b, t, hq, d), dtype=torch.float64), torch.zeros((b, t, hq, d), dtype=torch.float64)
    lse, reach = torch.full((b, t, hq), -math.inf, dtype=torch.float64), torch.zeros((b, t, hq), dtype=torch.float64)
    kp, vp, okp = cache.read(prefix_table, list(range(prefix_len)))
    for i in range(b):
        n = max(0, min(lens[i], len(tables[i]) * cache.bs))
        ko, vo, oko = cache.read(tables[i], list(range(n)))
        for step in range(t):
            m = max(0, n - t + step + 1)
            k, v = torch.cat([kp[okp], ko[:m][oko[:m]]]), torch.cat([vp[okp], vo[:m][oko[:m]]])  # [keys, h, d]
            if k.shape[0] == 0:
                continue
            rows = q[i, step].view(h, g, d)
            s = torch.einsum("hgd,nhd->hgn", rows, k) * scale
            reach[i, step] = (torch.einsum("hgd,nhd->hgn", rows.abs(), k.abs()) * abs(scale)).amax(-1).reshape(hq)
            lse[i, step] = torch.logsumexp(s, -1).reshape(hq)
            p = torch.softmax(s, -1)
            out[i, step] = torch.einsum("hgn,nhd->hgd", p, v).reshape(hq, d)
            mass[i, step] = torch.einsum("hgn,nhd->hgd", p, v.abs()).reshape(hq, d)
    return out, lse, mass, reach


def verify(target: torch.Tensor, draft: torch.Tensor | None, tokens: torch.Tensor, uniforms: torch.Tensor) -> tuple[list[int], list[int]]:
    """Kept counts and next tokens, sums by math.fsum."""
    kept, following = [], []
    b, k = tokens.shape
    vocab = target.shape[-1]
    for i in range(b):
        n, x = 0, -1
        while n < k:
            x = int(tokens[i, n])
            q = 1.0 if draft is None else (float(draft[i, n, x]) if 0 <= x < vocab else 0.0)
            if not 0 <= x < vocab or not float(uniforms[i, n]) * q < float(target[i, n, x]):
                break
            n += 1
        p = target[i, n].double().tolist()
        w = [max(a, 0.0) for a in p]
        if n < k and 0 <= x < vocab:
            left = [0.0 if v == x else max(a, 0.0) for v, a in enumerate(p)] if draft is None else [
                max(a - c, 0.0) for a, c in zip(p, draft[i, n].double().tolist())]
            if math.fsum(left) > 0:
                w = left
        total = math.fsum(w)
        kept.append(n)
        if not 0 < total < math.inf:
            following.append(-1)
            continue
        at, run, pick = float(uniforms[i, k]) * total, 0.0, -1
        for v, a in enumerate(w):
            run += a
            if run > at:
                pick = v
                break
        following.append(pick)
    return kept, following
