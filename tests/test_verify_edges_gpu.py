"""Draft verification where the border of two tokens falls on a rounding of its sums."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [20480, 20479])
def test_a_border_on_a_rounding_belongs_to_a_token_that_weighs_something(vocab: int) -> None:
    """Rows whose weights come twice, in the first half and, in another order, in the second: u = 1/2 is the border between
    the halves, on which sums in different orders differ by a bit. Weights lie far apart, with whole tiles of none between
    and behind them. The token drawn is one at which the cumulative sum passes the border, give or take 2^-48 of the total."""
    from lazykv_b200 import kernels as K

    gen = torch.Generator().manual_seed(3)
    b = 1200  # as many as have one CTA each, whose lanes take several tiles
    target = torch.zeros((b, 1, vocab))
    for i in range(b):
        n = int(torch.randint(3, 9, (1,), generator=gen))
        w = torch.rand(n, generator=gen) * 10 ** (-12 * torch.rand(n, generator=gen))
        for start, order in ((0, torch.arange(n)), (10240, torch.randperm(n, generator=gen))):
            at = start + torch.sort(torch.randperm(10, generator=gen)[:n])[0] * 1024 + torch.randint(0, 512, (n,), generator=gen)
            target[i, 0, at] = w[order]
    kept, token = K.verify_drafts(target.cuda(), None, torch.zeros((b, 0), dtype=torch.int64, device="cuda"), torch.full((b, 1), 0.5, device="cuda"))
    assert bool((kept == 0).all())
    for i, got in enumerate(token.tolist()):
        where = torch.nonzero(target[i, 0])[:, 0].tolist()
        w = target[i, 0, where].double().tolist()
        total = math.fsum(w)
        fine = [v for k, v in enumerate(where) if math.fsum(w[: k + 1]) >= total * (0.5 - 2.0**-48) and math.fsum(w[:k]) <= total * (0.5 + 2.0**-48)]
        assert got in fine, (i, got, fine)
