"""Draft verification on the GPU: kept counts and drawn tokens equal the definition's, and over many
draws the kept and drawn tokens together follow the target's probabilities."""

from __future__ import annotations

import pytest
import torch

from tests.paged_plain import verify

pytestmark = pytest.mark.gpu


def _case(gen: torch.Generator, b: int, k: int, v: int, noise: float = 0.5):
    logits = torch.randn((b, k + 1, v), generator=gen) * 2
    target = torch.softmax(logits, -1)
    draft = torch.softmax(logits[:, :k] + noise * torch.randn((b, k, v), generator=gen), -1)
    tokens = torch.multinomial(draft.reshape(b * k, v), 1, generator=gen).view(b, k) if k else torch.zeros((b, 0), dtype=torch.int64)
    return target, draft, tokens, torch.rand((b, k + 1), generator=gen)


def _same(target, draft, tokens, uniforms) -> None:  # noqa: ANN001
    from lazykv_b200 import kernels as K

    kept, token = K.verify_drafts(target.cuda(), None if draft is None else draft.cuda(), tokens.cuda(), uniforms.cuda())
    assert kept.dtype == torch.int32 and token.dtype == torch.int64
    want = verify(target, draft, tokens, uniforms)
    assert kept.tolist() == want[0] and token.tolist() == want[1]


@pytest.mark.parametrize("greedy", [False, True])
@pytest.mark.parametrize("b,k,v", [(1, 0, 5), (1, 1, 1), (4, 3, 7), (9, 8, 511), (3, 2, 512), (5, 4, 513), (2, 5, 8193), (1, 3, 100001), (150, 2, 1000), (3, 1, 131072), (320, 1, 9000)])
def test_matches_the_definition(b: int, k: int, v: int, greedy: bool) -> None:
    gen = torch.Generator().manual_seed(b * 100 + v)
    target, draft, tokens, uniforms = _case(gen, b, k, v)
    _same(target, None if greedy else draft, tokens, uniforms)


def test_a_vocabulary_of_more_tiles_than_one_cta_keeps() -> None:
    gen = torch.Generator().manual_seed(4)
    b, k, v = 300, 1, 600_000  # 300 sequences would have one CTA each; 600,000 elements are more than its 1,024 tile sums
    target = torch.rand((1, k + 1, v), generator=gen)
    uniforms = torch.rand((b, k + 1), generator=gen)
    uniforms[:, 0] = 0.9999
    tokens = torch.randint(0, v, (b, k), generator=gen)
    from lazykv_b200 import kernels as K

    kept, token = K.verify_drafts(target.cuda().expand(b, k + 1, v), None, tokens.cuda(), uniforms.cuda())
    edges = [torch.cumsum(target[0, i].double(), 0) for i in range(2)]
    for i in range(b):
        n = int(0.9999 < 0 or float(uniforms[i, 0]) < float(target[0, 0, int(tokens[i, 0])]))
        assert int(kept[i]) == n
        e = edges[n].clone()
        if n == 0:
            w = target[0, 0].double().clone()
            w[int(tokens[i, 0])] = 0
            e = torch.cumsum(w, 0)
        assert int(token[i]) == int(torch.searchsorted(e, float(uniforms[i, 1]) * e[-1], right=True))


def test_borders_are_exact() -> None:
    """Dyadic probabilities, whose sums carry no rounding: u on a border belongs to the token above it."""
    target = torch.tensor([[[0.25, 0.0, 0.5, 0.25], [0.0, 0.0, 0.5, 0.5]]]).expand(6, 2, 4).contiguous()
    draft = torch.tensor([[[0.5, 0.25, 0.25, 0.0]]]).expand(6, 1, 4).contiguous()
    tokens = torch.tensor([[0], [0], [1], [2], [2], [3]])
    below, half = 0.5 - 2.0**-25, 0.5
    uniforms = torch.tensor([[below, 0.0], [half, 0.0], [0.0, 0.5], [1 - 2.0**-24, 0.5], [0.3, 0.5 - 2.0**-25], [0.999, 0.999]])
    # row 1: u q = 0.25 is not below p = 0.25; row 2: p = 0 keeps nothing, even at u = 0
    _same(target, draft, tokens, uniforms)
    from lazykv_b200 import kernels as K

    kept, token = K.verify_drafts(target.cuda(), draft.cuda(), tokens.cuda(), uniforms.cuda())
    # residual of the first row: [0, 0, 0.25, 0.25]
    assert kept.tolist() == [1, 0, 0, 1, 1, 1] and token.tolist() == [2, 2, 3, 3, 2, 3]


def test_ended_drafts_equal_rows_and_weightless_rows() -> None:
    gen = torch.Generator().manual_seed(11)
    target, draft, tokens, uniforms = _case(gen, 8, 3, 300)
    uniforms[:, :3] = 0.0  # everything with a positive probability is kept
    tokens[0, 0] = -1
    tokens[1, 2] = -1
    tokens[2, 1] = 300  # outside the vocabulary
    draft[3] = target[3, :3]
    target[4, 0] = 0.0  # rejected, and nothing to draw from
    target[5, 3] = 0.0
    target[5, 3, 299] = 2.0**-140  # one token with a subnormal weight
    target[6, 0, 7] = torch.nan  # a NaN weighs nothing
    uniforms[7, 0] = 0.99999994
    _same(target, draft, tokens, uniforms)
    from lazykv_b200 import kernels as K

    # where the draft's row equals the target's and the token is refused, the target's own row is drawn from
    t = torch.tensor([[[0.5, 0.5, 0.0], [1.0, 0.0, 0.0]]])
    kept, token = K.verify_drafts(t.cuda(), t[:, :1].contiguous().cuda(), torch.tensor([[2]]).cuda(), torch.tensor([[0.0, 0.75]]).cuda())
    assert kept.tolist() == [0] and token.tolist() == [1]
    t[0, 0] = torch.inf
    kept, token = K.verify_drafts(t.cuda(), None, torch.tensor([[-1]]).cuda(), torch.tensor([[0.0, 0.75]]).cuda())
    assert kept.tolist() == [0] and token.tolist() == [-1]


def test_strided_rows_and_a_graph() -> None:
    from lazykv_b200 import kernels as K

    gen = torch.Generator().manual_seed(12)
    b, k, v = 5, 4, 1001
    target, draft, tokens, uniforms = _case(gen, b, k, v)
    want = verify(target, draft, tokens, uniforms)
    wide = torch.full((b, k + 1, v + 30), 9.0, device="cuda")
    wide[..., 3 : v + 3] = target.cuda()
    wide_q = torch.full((b, k, 2 * v), 9.0, device="cuda")
    wide_q[..., 1 : v + 1] = draft.cuda()
    toks = torch.full((b, k + 5), -1, device="cuda")
    toks[:, :k] = tokens.cuda()
    u = uniforms.cuda()
    args = (wide[..., 3 : v + 3], wide_q[..., 1 : v + 1], toks[:, :k], u)
    kept, token = K.verify_drafts(*args)
    assert kept.tolist() == want[0] and token.tolist() == want[1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, token = K.verify_drafts(*args)
    u.copy_(torch.rand((b, k + 1), generator=gen))
    graph.replay()
    want = verify(target, draft, tokens, u.cpu())
    assert kept.tolist() == want[0] and token.tolist() == want[1]


def test_kept_and_drawn_tokens_follow_the_target() -> None:
    """The first emitted token of 200,000 independent runs: its counts are within 5 standard deviations of
    the target's probabilities, for every token (the draft's own are off by far more)."""
    from lazykv_b200 import kernels as K

    gen = torch.Generator(device="cuda").manual_seed(13)
    n, v = 200_000, 6
    p = torch.tensor([0.05, 0.4, 0.1, 0.25, 0.15, 0.05], device="cuda")
    q = torch.tensor([0.3, 0.1, 0.3, 0.1, 0.1, 0.1], device="cuda")
    tokens = torch.multinomial(q, n, replacement=True, generator=gen).view(n, 1)
    target = torch.stack([p, p.flip(0)]).expand(n, 2, v)
    kept, token = K.verify_drafts(target, q.expand(n, 1, v), tokens, torch.rand((n, 2), generator=gen, device="cuda"))
    first = torch.where(kept > 0, tokens[:, 0], token)
    count = torch.bincount(first, minlength=v).double().cpu()
    pd = p.double().cpu()
    assert bool(((count - n * pd).abs() <= 5 * (n * pd * (1 - pd)).sqrt()).all()), (count / n).tolist()
